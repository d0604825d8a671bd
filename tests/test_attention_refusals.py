"""CPU: the entry points of the attention block return their codes before any HIP call (the
pointers here are never dereferenced), and the Python layer names what is wrong."""
import os

import pytest
import torch

from ferret_amd import lib

P = 1 << 20  # aligned, never read


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    return lib.load()


def _swap(args, **changes):
    out = list(args)
    for at, v in changes.items():
        out[int(at[1:])] = v
    return out


def test_norm(L):
    #       x  stride   r  stride w  eps  M  K     y       r_out stream
    good = [P, 4096, 2 * P, 4096, P // 2, 1e-6, 4, 4096, 3 * P, 4 * P, None]
    f = L.ferret_rms_norm
    for at, v, rc in [(0, None, -1), (2, None, -1), (4, None, -1), (8, None, -1), (9, None, -1), (6, 0, -2), (7, 0, -2),
                      (7, 4100, -2), (7, 65536, -2), (5, -1e-6, -2), (5, float("nan"), -2), (5, float("inf"), -2),
                      (1, 4088, -2), (0, P + 8, -4), (1, 4100, -4), (3, 4097, -4), (4, P // 2 + 2, -4), (8, 3 * P + 8, -4),
                      (8, P + 16, -2), (9, 2 * P + 4096, -2), (9, 3 * P, -2), (8, P // 2, -2)]:
        assert f(*_swap(good, **{f"_{at}": v})) == rc, (at, v)
    g = L.ferret_rms_norm_e4m3  # ..., q, scale, residual_out, stream
    good8 = [P, 4096, None, 0, P // 2, 1e-6, 4, 4096, 3 * P, 4 * P, None, None]
    for at, v, rc in [(9, None, -1), (8, None, -1), (7, 4104, -2), (8, 3 * P + 4, -4), (9, 4 * P + 2, -4), (8, P, -2),
                      (9, 3 * P, -2), (9, P + 64, -2)]:
        assert g(*_swap(good8, **{f"_{at}": v})) == rc, (at, v)


def test_cache(L):
    #       latent    rotary    table lens cu B pages T  data scales pages page stream
    good = [P, 512, 2 * P, 64, P, P, P, 3, 8, 5, 4 * P, 5 * P, 100, 64, None]
    f = L.ferret_latent_cache_write
    for at, v, rc in [(0, None, -1), (2, None, -1), (4, None, -1), (5, None, -1), (6, None, -1), (10, None, -1), (7, 0, -2),
                      (8, 0, -2), (9, 0, -2), (12, 0, -2), (13, 8, -2), (13, 40, -2), (13, 0, -2), (8, 1 << 26, -2),
                      (1, 504, -2), (3, 56, -2), (0, P + 2, -4), (1, 516, -4), (3, 68, -4), (10, 4 * P + 8, -4),
                      (11, 5 * P + 1, -4)]:
        assert f(*_swap(good, **{f"_{at}": v})) == rc, (at, v)
    #       data scales pages page table cu B pages rows latent rotary stream
    good = [P, None, 100, 64, P, P, 3, 8, 50, 2 * P, 3 * P, None]
    g = L.ferret_latent_cache_read
    for at, v, rc in [(0, None, -1), (4, None, -1), (5, None, -1), (9, None, -1), (10, None, -1), (8, 0, -2), (3, 24, -2),
                      (2, 0, -2), (6, 0, -2), (9, 2 * P + 8, -4)]:
        assert g(*_swap(good, **{f"_{at}": v})) == rc, (at, v)


def test_absorbed(L):
    need = L.ferret_latent_attention_workspace(3, 5, 16)
    assert need > 0 and L.ferret_latent_attention_workspace(0, 5, 16) == 0
    assert L.ferret_latent_attention_workspace(1, 1 << 20, 1 << 20) == 0
    #       ql    t     h    qr  t     h   data scales pages page table lens cu B mp T  H  scale causal out lse ws bytes st
    good = [P, 8192, 512, P, 1024, 64, P, P, 100, 64, P, P, P, 3, 8, 5, 16, 0.07, 1, P, None, P, need, None]
    f = L.ferret_latent_attention
    for at, v, rc in [(0, None, -1), (3, None, -1), (6, None, -1), (10, None, -1), (11, None, -1), (12, None, -1),
                      (19, None, -1), (13, 0, -2), (14, 0, -2), (15, 0, -2), (16, 0, -2), (16, 1025, -2), (9, 17, -2),
                      (17, 0.0, -2), (17, -1.0, -2), (17, float("nan"), -2), (17, float("inf"), -2), (1, -8, -2),
                      (2, 1 << 31, -2), (21, None, -3), (22, need - 1, -3), (21, P + 4, -3), (0, P + 2, -4), (1, 8196, -4),
                      (5, 60, -4), (19, P + 8, -4), (20, P + 2, -4), (7, P + 1, -4), (14, 1 << 25, -2)]:
        assert f(*_swap(good, **{f"_{at}": v})) == rc, (at, v)


def test_expanded(L):
    #       qn    t     h    qr   t    h   kn   s     h   kr  s   v   s     h   cu cu B  T  S  H scale causal out lse ws bytes st
    good = [P, 3008, 192, P, 3008, 192, P, 4096, 256, P, 64, P, 4096, 256, P, P, 2, 9, 30, 16, 0.07, 1, P, None, None, 0,
            None]
    f = L.ferret_latent_attention_expanded
    for at, v, rc in [(0, None, -1), (3, None, -1), (6, None, -1), (9, None, -1), (11, None, -1), (14, None, -1),
                      (15, None, -1), (22, None, -1), (16, 0, -2), (17, 0, -2), (18, 0, -2), (19, 0, -2), (19, 1025, -2),
                      (20, 0.0, -2), (20, float("nan"), -2), (7, 1 << 24, -2), (10, -8, -2), (1, 3010, -4), (13, 260, -4),
                      (6, P + 4, -4), (22, P + 2, -4), (23, P + 1, -4)]:
        assert f(*_swap(good, **{f"_{at}": v})) == rc, (at, v)
    need = L.ferret_latent_attention_expanded_workspace(2, 9, 8000, 16)
    assert need == 8 * 9 * 16 * (8 + 512) and L.ferret_latent_attention_expanded_workspace(2, 9, 30, 16) == 0
    assert L.ferret_latent_attention_expanded_workspace(0, 9, 8000, 16) == 0
    split = _swap(good, _18=8000, _24=P, _25=need)
    for at, v in [(24, None), (24, P + 8), (25, need - 1)]:
        assert f(*_swap(split, **{f"_{at}": v})) == -3, (at, v)


def test_python_layer_refuses_cpu_tensors_and_other_caches():
    from ferret_amd import ops
    bf = dict(dtype=torch.bfloat16)
    x, w = torch.zeros((2, 128), **bf), torch.zeros(128, **bf)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_e4m3(x, w),
                 lambda: ops.latent_cache_read(ops.LatentCache.empty(1, 16, device="cpu"),
                                               torch.zeros((1, 1), dtype=torch.int32),
                                               torch.zeros(2, dtype=torch.int32), 1)):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    q = torch.zeros((1, 2, 512), **bf)
    with pytest.raises(TypeError, match="LatentCache"):
        ops.latent_attention(q, q, q, q, q, q, 1.0)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.latent_attention_expanded(q[..., :128], q[..., :64], q[..., :128], q[0, :, :64], q[..., :128], q, q, 1.0)
    with pytest.raises(ValueError, match="bf16 or e4m3"):
        ops.LatentCache.empty(1, 16, torch.float32, device="cpu")


def test_fake_shapes():
    import ferret_amd.torch_ops  # noqa: F401
    T = torch.ops.ferret

    def m(*s, dtype=torch.bfloat16):
        return torch.empty(s, dtype=dtype, device="meta")
    i32 = torch.int32
    assert T.rms_norm(m(5, 512), m(512)).shape == (5, 512)
    y, r = T.add_rms_norm(m(5, 512), m(5, 512), m(512))
    assert y.dtype == r.dtype == torch.bfloat16
    q, s = T.rms_norm_e4m3(m(5, 512), m(512))
    assert q.dtype == torch.float8_e4m3fn and s.shape == (5, 4) and s.dtype == torch.float32
    assert T.add_rms_norm_e4m3(m(5, 512), m(5, 512), m(512))[2].shape == (5, 512)
    data, scales = m(7, 64, 640, dtype=torch.uint8), m(7, 64, 4, dtype=torch.uint8)
    T.latent_cache_write(data, scales, m(3, 512), m(3, 64), m(2, 4, dtype=i32), m(2, dtype=i32), m(3, dtype=i32))
    lat, rot = T.latent_cache_read(data, scales, m(2, 4, dtype=i32), m(3, dtype=i32), 90)
    assert lat.shape == (90, 512) and rot.shape == (90, 64)
    o, lse = T.latent_attention(m(3, 16, 512), m(3, 16, 64), data, scales, m(2, 4, dtype=i32), m(2, dtype=i32),
                                m(3, dtype=i32), 0.1)
    assert o.shape == (3, 16, 512) and lse.shape == (3, 16) and lse.dtype == torch.float32
    o, lse = T.latent_attention_expanded(m(3, 16, 128), m(3, 16, 64), m(9, 16, 128), m(9, 64), m(9, 16, 128),
                                         m(3, dtype=i32), m(3, dtype=i32), 0.1)
    assert o.shape == (3, 16, 128) and lse.shape == (3, 16)
