"""CPU: the int8 entry points and the attention over shared prefixes return their codes before any HIP
call (the pointers here are never dereferenced), and the Python layer names what is wrong."""
import os

import pytest
import torch

from ferret_amd import lib

P = 1 << 24  # aligned, never read


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    return lib.load()


def _refused(f, good, wrong):
    for at, v, rc in wrong:
        args = list(good)
        args[at] = v
        assert f(*args) == rc, (at, v)


def test_quantizer(L):
    #       x  stride M  K     q      scale  stream
    good = [P, 4096, 4, 4096, 2 * P, 3 * P, None]
    _refused(L.ferret_quant_act_int8, good, [
        (0, None, -1), (4, None, -1), (5, None, -1), (2, 0, -2), (3, 0, -2), (3, 8, -2), (3, 4104, -2), (3, 32784, -2),
        (1, 4088, -2), (1, 0, -2), (1, -4096, -2), (0, P + 8, -4), (1, 4100, -4), (4, 2 * P + 8, -4), (5, 3 * P + 2, -4),
        (4, P, -2), (4, P + 16, -2), (5, P + 64, -2), (5, 2 * P, -2)])


def test_product(L):
    #       a   sa     b      sb     r     y      M   N     K    ws  bytes stream
    good = [P, 2 * P, 3 * P, 8 * P, None, 9 * P, 16, 4096, 4096, None, 0, None]
    assert L.ferret_int8_gemm_workspace(0, 4096, 4096) == 0 and L.ferret_int8_gemm_workspace(16, 4100, 4096) == 0
    f = L.ferret_int8_gemm
    _refused(f, good, [
        (0, None, -1), (1, None, -1), (2, None, -1), (3, None, -1), (5, None, -1), (6, 0, -2), (7, 0, -2), (7, 4092, -2),
        (8, 0, -2), (8, 4088, -2), (8, 65552, -2), (0, P + 8, -4), (1, 2 * P + 2, -4), (2, 3 * P + 4, -4), (3, 8 * P + 4, -4),
        (4, 10 * P + 8, -4), (5, 9 * P + 8, -4)])
    big = [P, 2 * P, 3 * P, 8 * P, None, 9 * P, 16, 4096, 12288, 10 * P, L.ferret_int8_gemm_workspace(16, 4096, 12288),
           None]
    if big[10]:
        _refused(f, big, [(9, None, -3), (10, big[10] - 1, -3), (9, 10 * P + 8, -3), (9, 9 * P, -2), (9, 3 * P, -2)])
    # outputs over what is read, and over the residual elsewhere than in place
    need = L.ferret_int8_gemm_workspace(16, 4096, 4096)
    small = good[:9] + [20 * P, need, None]
    _refused(f, small, [(5, P, -2), (5, 2 * P, -2), (5, 3 * P + 16, -2), (5, 8 * P, -2), (4, 9 * P + 16, -2)])


def test_shared(L):
    need = L.ferret_latent_attention_shared_workspace(2, 3, 5, 16)
    assert need > 0 and L.ferret_latent_attention_shared_workspace(0, 3, 5, 16) == 0
    assert L.ferret_latent_attention_shared_workspace(2, 0, 5, 16) == 0
    assert L.ferret_latent_attention_shared_workspace(1, 1, 1 << 20, 1 << 20) == 0
    Q, R, D, S, X, O, W = (i * P for i in (1, 2, 3, 5, 6, 7, 8))
    #       ql t     h    qr t     h  data sc pages page ptab plens cup  G  mpp tab  lens  cu   B  mp T  H scale
    good = [Q, 8192, 512, R, 1024, 64, D, S, 100, 64, X, X + 64, X + 128, 2, 8, X + 512, X + 1024, X + 1088, 3, 8, 5, 16, 0.07,
            1, O, None, W, need, None]  # causal out lse ws bytes stream
    _refused(L.ferret_latent_attention_shared, good, [
        (0, None, -1), (3, None, -1), (6, None, -1), (10, None, -1), (11, None, -1), (12, None, -1), (15, None, -1),
        (16, None, -1), (17, None, -1), (24, None, -1), (13, 0, -2), (14, 0, -2), (18, 0, -2), (19, 0, -2), (20, 0, -2),
        (21, 0, -2), (21, 1025, -2), (9, 17, -2), (22, 0.0, -2), (22, float("nan"), -2), (22, float("inf"), -2), (1, -8, -2),
        (2, 1 << 31, -2), (26, None, -3), (27, need - 1, -3), (26, W + 4, -3), (0, Q + 2, -4), (1, 8196, -4), (5, 60, -4),
        (24, O + 8, -4), (25, O + 2, -4), (7, S + 1, -4), (14, 1 << 25, -2), (19, 1 << 25, -2),
        # outputs and workspace over what is read
        (24, R, -2), (24, D + 64, -2), (24, X, -2), (24, Q + 16, -2), (25, X + 128, -2), (26, D, -2), (26, O, -2),
        (26, X + 1024, -2), (25, O + 64, -2)])


def test_sizes_past_a_launch(L):
    """Rows, tiles and query rows whose launch would pass 2^32 threads."""
    far = 1 << 45  # no range ends in another
    assert L.ferret_quant_act_int8(P, 64, 1 << 22, 64, far, 2 * far, None) == -2
    for m, n in ((1 << 22, 64), (64, 1 << 22), ((1 << 22) - 8, (1 << 22) - 8)):
        assert L.ferret_int8_gemm_workspace(m, n, 64) == 0
        assert L.ferret_int8_gemm(P, far, 2 * far, 3 * far, None, 4 * far, m, n, 64, None, 0, None) == -2
    T, ws = 1 << 20, L.ferret_latent_attention_shared_workspace
    assert ws(1, 1, T, 64) == 0 and ws(1, 1, T - 1, 64) > 0 and ws(1, 1 << 26, 1, 1) == 0
    assert L.ferret_latent_attention_shared(
        P, 64 * 512, 512, far, 64 * 64, 64, 2 * far, None, 100, 64, 3 * far, 3 * far + 512, 3 * far + 1024, 1, 8,
        3 * far + 1536, 3 * far + 2048, 3 * far + 2560, 1, 8, T, 64, 0.07, 1, 4 * far, None, 5 * far, far, None) == -2


def test_python_names_what_is_wrong():
    from ferret_amd import ops
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    i = torch.zeros((2, 128), dtype=torch.int8)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.quant_act_int8(x)
    with pytest.raises(ValueError, match="2-D"):
        ops.quant_act_int8(x[0])
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.int8_gemm(i, torch.ones(2), i, torch.ones(2))
    with pytest.raises(TypeError, match="LatentCache"):
        ops.latent_attention_shared(x, x, None, x, x, x, x, x, x, 0.1)
    cache = ops.LatentCache(torch.zeros((4, 16, 576), dtype=torch.bfloat16))
    t = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.latent_attention_shared(x, x, cache, t, t[0, :1], t[0, :2], t, t[0, :1], t[0, :2], 0.1)


def test_fake_shapes():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    import ferret_amd.torch_ops  # noqa: F401
    F, m = torch.ops.ferret, lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="meta")
    bf, i8, i32 = torch.bfloat16, torch.int8, torch.int32
    q, s = F.quant_act_int8(m(33, 4096, dtype=bf))
    assert q.shape == (33, 4096) and q.dtype == i8 and s.shape == (33,) and s.dtype == torch.float32
    y = F.int8_gemm(m(33, 4096, dtype=i8), m(33), m(6144, 4096, dtype=i8), m(6144), m(33, 6144, dtype=bf))
    assert y.shape == (33, 6144) and y.dtype == bf
    o, lse = F.latent_attention_shared(m(5, 16, 512, dtype=bf), m(5, 16, 64, dtype=bf), m(9, 64, 576, dtype=bf), None,
                                       m(1, 4, dtype=i32), m(1, dtype=i32), m(2, dtype=i32), m(3, 4, dtype=i32),
                                       m(3, dtype=i32), m(4, dtype=i32), 0.07)
    assert o.shape == (5, 16, 512) and o.dtype == bf and lse.shape == (5, 16)
