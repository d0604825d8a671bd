"""CPU: sizes past 2^31 are refused where they meet the C ABI's ints, which would take their low 32 bits."""
import ctypes
import os

import pytest
import torch

from ferret_amd import lib, ops

FAR = (1 << 32) + 20  # its low 32 bits are 20


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    return lib.load()


def test_sizes_of_workspaces(L):
    assert ops.int8_gemm_workspace_bytes(20, 520, 4096) > 0
    for m, n, k in ((FAR, 520, 4096), (20, (1 << 32) + 520, 4096), (20, 520, (1 << 32) + 4096)):
        with pytest.raises((ValueError, ctypes.ArgumentError), match="32 bits"):
            ops.int8_gemm_workspace_bytes(m, n, k)
    with pytest.raises((ValueError, ctypes.ArgumentError), match="32 bits"):
        ops.latent_attention_shared_workspace_bytes(1, 4, FAR, 16)
    with pytest.raises((ValueError, ctypes.ArgumentError), match="32 bits"):
        ops.latent_attention_workspace_bytes(4, FAR, 16)
    assert L.ferret_int8_gemm_workspace(-1, 520, 4096) == 0       # negative numbers are the library's to refuse


def test_tensors_of_many_rows():
    """Such tensors fit the GPU: 2^32 rows of 16 codes are 64 GiB."""
    sa, sb = meta(20, dtype=torch.float32), meta(32, dtype=torch.float32)
    few, many = meta(32, 16, dtype=torch.int8), meta(FAR, 16, dtype=torch.int8)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.quant_act_int8(meta(FAR, 16))
    with pytest.raises(ValueError, match="2\\^31"):
        ops.int8_gemm(many, sa, few, sb)
    with pytest.raises(ValueError, match="2\\^31"):
        ops._dev(many, "b", torch.int8, 2)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.linear_bf16(meta(FAR, 16), meta(32, 16))
    with pytest.raises(ValueError, match="2\\^31"):
        ops.rms_norm(meta(FAR, 16), meta(16))
