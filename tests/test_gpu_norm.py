"""GPU: rms_norm and rms_norm_e4m3 against the formula in 64 bits.

Bounds: the kernel's fp32 steps (a sum of K squares in registers, its root, three
products) are off by at most (K/64 + 16) * 2^-24 relative in the sum's chain and a few
steps after it, below 2^-13 for K <= 32768; a bf16 result adds half a step, 2^-8
of the value; an e4m3 code half of its step: 2^-4 of the value, or 2^-10 of the scale
for the codes below 2^-6.  A scale adds two fp32 roundings.
"""
import numpy as np
import pytest
import torch

from oracle import attention as A
from tests.attention_helpers import bf16_tensor, bf16_values

pytestmark = pytest.mark.gpu
FP32 = 2.0 ** -13


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


def _case(M, K, res, wide, seed=0):
    rng = np.random.default_rng(seed + M + K)
    x = bf16_values(rng, M, K + wide)
    w = 1 + 0.3 * bf16_values(rng, K)
    w = bf16_tensor(w)
    r = bf16_values(rng, M, K, std=3.0) if res else None
    xt = bf16_tensor(x)[:, wide:]
    return x[:, wide:], xt, w, r, bf16_tensor(r) if res else None


SHAPES = [(1, 8), (3, 24), (5, 128), (64, 512), (7, 520), (33, 1024), (9, 1536), (2, 2048), (6, 2056), (5, 4096),
          (17, 7168), (3, 7176), (2, 16384), (2, 24576), (3, 32768)]


@pytest.mark.parametrize("M,K", SHAPES)
@pytest.mark.parametrize("res", [False, True])
def test_bf16(ops, M, K, res):
    print(f"[case] rms_norm M={M} K={K} residual={res}", flush=True)
    x, xt, w, r, rt = _case(M, K, res, 16 if K % 3 else 0)
    y, ro = ops.rms_norm(xt, w, rt, eps=1e-5)
    torch.cuda.synchronize()
    want, s = A.rms_norm(x, w.float().cpu().numpy(), r, 1e-5)
    got = y.float().cpu().numpy()
    assert (np.abs(got - want) <= (2.0 ** -8 + FP32) * np.abs(want) + 1e-38).all()
    if res:
        assert torch.equal(ro, (xt.float() + rt.float()).to(torch.bfloat16))
    else:
        assert ro is None


@pytest.mark.parametrize("M,K", [s for s in SHAPES if s[1] % 128 == 0])
@pytest.mark.parametrize("res", [False, True])
def test_e4m3(ops, M, K, res):
    print(f"[case] rms_norm_e4m3 M={M} K={K} residual={res}", flush=True)
    x, xt, w, r, rt = _case(M, K, res, 8, seed=9)
    if M > 2:  # a block of zeros (the floor of the scale) and one of tiny values (codes below 2^-6)
        for t in (x, r):
            if t is not None:
                t[1, :128] = 0
                t[2, -128:] *= 2.0 ** -12
        xt = bf16_tensor(np.concatenate([np.zeros((M, 8), np.float32), x], 1))[:, 8:]
        rt = bf16_tensor(r) if res else None
    q, scale, ro = ops.rms_norm_e4m3(xt, w, rt)
    torch.cuda.synchronize()
    want, _ = A.rms_norm(x, w.float().cpu().numpy(), r, 1e-6)
    amax = np.maximum(np.abs(want).reshape(M, -1, 128).max(-1), 1e-4)
    sc = scale.cpu().numpy().astype(np.float64)
    assert (np.abs(sc - amax / 448) <= (FP32 + 2.0 ** -23) * amax / 448).all()
    got = q.float().cpu().numpy().astype(np.float64) * sc.repeat(128, 1)
    assert (np.abs(got - want) <= (2.0 ** -4 + 2 * FP32) * np.abs(want) + 2.0 ** -10 * sc.repeat(128, 1)).all()
    if res:
        assert torch.equal(ro, (xt.float() + rt.float()).to(torch.bfloat16))


def test_e4m3_feeds_the_fp8_product(ops):
    """The codes and scales of the norm are what fp8_gemm_blockscale takes."""
    from ferret_amd import workloads as W
    print("[case] norm into the FP8 product", flush=True)
    x, xt, w, _, _ = _case(40, 1536, False, 576)
    q, scale, _ = ops.rms_norm_e4m3(xt, w)
    b, sb = W.quant_weight_128x128(W.randn((256, 1536), 4, "cuda"))
    c = ops.fp8_gemm_blockscale(q, scale, b, sb).float()
    a = q.float().cpu().double() * scale.cpu().double().repeat_interleave(128, 1)
    bf = b.float().cpu().double() * sb.cpu().double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    ref = a @ bf.T
    torch.cuda.synchronize()
    bound = 2.0 ** -8 * ref.abs() + 1536 * 2.0 ** -23 * (a.abs() @ bf.abs().T)
    assert ((c.cpu().double() - ref).abs() <= bound).all()


def test_in_place_gives_the_same_bits(ops):
    print("[case] rms_norm in place", flush=True)
    _, xt, w, _, rt = _case(300, 7168, True, 0)
    y, ro = ops.rms_norm(xt, w, rt)
    x2, r2 = xt.clone(), rt.clone()
    a, b = ops.rms_norm(x2, w, r2, out=x2, residual_out=r2)
    assert a is x2 and b is r2 or (a.data_ptr() == x2.data_ptr() and b.data_ptr() == r2.data_ptr())
    assert torch.equal(x2, y) and torch.equal(r2, ro)


def test_rows_of_zeros_inf_and_nan_stay_their_own(ops):
    print("[case] rms_norm special rows", flush=True)
    _, xt, w, _, _ = _case(6, 512, False, 0)
    clean = ops.rms_norm(xt, w)[0]
    x = xt.clone()
    x[1] = 0
    x[3, 7] = float("nan")
    x[4, 500] = float("inf")
    y = ops.rms_norm(x, w)[0]
    q, s, _ = ops.rms_norm_e4m3(x, w)
    torch.cuda.synchronize()
    assert torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]])
    assert (y[1] == 0).all() and y[3].isnan().all()
    assert y[4, 500].isnan() and (y[4, :500] == 0).all()     # 1 / sqrt(inf) = 0, inf * 0
    assert (q[1].float() == 0).all() and (s[1] == torch.tensor(1e-4) / 448).all()
    assert q[3].float().isnan().all() and torch.isfinite(s).all()


def test_refusals(ops):
    _, xt, w, _, rt = _case(4, 512, True, 0)
    with pytest.raises(TypeError):
        ops.rms_norm(xt.float(), w)
    with pytest.raises(ValueError, match="w must be"):
        ops.rms_norm(xt, w[:256])
    with pytest.raises(ValueError, match="residual_out needs"):
        ops.rms_norm(xt, w, residual_out=rt)
    with pytest.raises(ValueError, match="residual must be"):
        ops.rms_norm(xt, w, rt[:2])
    with pytest.raises(ValueError, match="16-byte bound"):
        ops.rms_norm(torch.zeros((4, 516), dtype=torch.bfloat16, device="cuda")[:, 4:], w)   # 8 bytes off
    with pytest.raises(ValueError, match="16-byte bound"):
        ops.rms_norm(torch.zeros((4, 515), dtype=torch.bfloat16, device="cuda")[:, :512], w)  # stride 515
    with pytest.raises(ValueError, match="packed"):
        ops.rms_norm(torch.zeros((512, 4), dtype=torch.bfloat16, device="cuda").t(), w)
    with pytest.raises(RuntimeError, match="code -2"):   # overlapping, but not in place
        ops.rms_norm(xt[:3], w, out=xt[1:])
    with pytest.raises(RuntimeError, match="code -2"):   # e4m3 needs whole blocks
        ops.rms_norm_e4m3(xt[:, :264].contiguous(), w[:264].contiguous())
    with pytest.raises(RuntimeError, match="code -2"):
        ops.rms_norm(xt, w, eps=-1.0)
    with pytest.raises(RuntimeError, match="code -2"):
        ops.rms_norm(xt, w, eps=float("nan"))


def test_captured_and_replayed(ops):
    print("[case] rms_norm graph", flush=True)
    _, xt, w, _, rt = _case(48, 2048, True, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rms_norm_e4m3(xt, w, rt)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.rms_norm_e4m3(xt, w, rt)
    for k in range(3):
        xt.copy_(torch.randn(xt.shape, device="cuda") * (k + 1))
        g.replay()
        want = ops.rms_norm_e4m3(xt, w, rt)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), k
