"""CPU: the row strides that the norms and the cache write hand to the library are the tensors' own.

The tensors here are host tensors that call themselves GPU ones, and the library is a recorder: what the
Python layer would launch is looked at, nothing is launched.
"""
import contextlib
import os

import pytest
import torch

from ferret_amd import lib, ops


class OnGpu(torch.Tensor):
    device = property(lambda self: torch.device("cuda", 0))


def gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnGpu)


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def recorded(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(lib, "load", lambda: rec)
    monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    monkeypatch.setattr(ops, "_on", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    return rec.calls


def _norm(x, r=None):
    M, K = x.shape
    ops.rms_norm(x, gpu(K), r, out=gpu(M, K), residual_out=None if r is None else gpu(M, K))


def _norm8(x, r=None):
    M, K = x.shape
    ops.rms_norm_e4m3(x, gpu(K), r, q=gpu(M, K, dtype=ops.FP8), scale=gpu(M, K // 128, dtype=torch.float32),
                      residual_out=None if r is None else gpu(M, K))


def _write(latent, rotary):
    i32 = torch.int32
    ops.latent_cache_write(ops.LatentCache(gpu(3, 16, 576)), latent, rotary, gpu(1, 3, dtype=i32), gpu(1, dtype=i32),
                           gpu(2, dtype=i32))


@pytest.mark.parametrize("norm", [_norm, _norm8])
def test_norms_refuse_rows_that_share_storage(recorded, norm):
    """Many rows of one row's storage: a stride of 0, which is no row pitch, nor is any below K."""
    for rows in (gpu(1, 512).expand(64, 512), gpu(64 * 512).as_strided((64, 512), (256, 1))):
        with pytest.raises(ValueError, match="x's rows"):
            norm(rows)
        with pytest.raises(ValueError, match="residual's rows"):
            norm(gpu(64, 512), rows)
    assert recorded == []


def test_cache_write_refuses_rows_that_share_storage(recorded):
    with pytest.raises(ValueError, match="latent's rows"):
        _write(gpu(1, 512).expand(8, 512), gpu(8, 64))
    with pytest.raises(ValueError, match="rotary's rows"):
        _write(gpu(8, 512), gpu(1, 64).expand(8, 64))
    assert recorded == []


def test_strides_are_handed_on(recorded):
    """Packed rows, slices of wider ones, and one row of any stride."""
    for x, stride in ((gpu(4, 512), 512), (gpu(4, 704)[:, 64:576], 704), (gpu(1, 704)[:, 64:576], 512),
                      (gpu(512).expand(1, 512), 512)):
        M = x.shape[0]
        _norm(x, x)
        _norm8(x, x)
        _write(x, gpu(M, 64))
        (_, a), (_, b), (_, c) = recorded[-3:]
        assert (a[1], a[3], b[1], b[3], c[1], c[3]) == (stride,) * 5 + (64,)


def test_the_library_refuses_a_stride_of_zero():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    L, P = lib.load(), 1 << 20   # never read
    for at in (1, 3):
        args = [P, 512, 2 * P, 512, P // 2, 1e-6, 64, 512, 3 * P, 4 * P, None]
        args[at] = 0
        assert L.ferret_rms_norm(*args) == -2
        args = [P, 512, 2 * P, 512, P // 2, 1e-6, 64, 512, 3 * P, 4 * P, 5 * P, None]
        args[at] = 0
        assert L.ferret_rms_norm_e4m3(*args) == -2
        args = [P, 512, 2 * P, 64, P, P, P, 1, 3, 8, 4 * P, None, 3, 16, None]
        args[at] = 0
        assert L.ferret_latent_cache_write(*args) == -2
