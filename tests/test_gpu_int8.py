"""The int8 quantizer and product on the GPU, bit for bit against the oracle."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ferret_amd import lib, ops
from oracle import formats as F
from oracle import int8 as I

pytestmark = pytest.mark.gpu


def bf16_tensor(x: np.ndarray) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).cuda()


def bits(t: torch.Tensor) -> np.ndarray:
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def rows_of(rng, M, K):
    size = np.exp2(rng.integers(-6, 7, (M, 1)))
    return F.bf16_round((rng.standard_normal((M, K)) * size).astype(np.float32))


def check_quant(x: np.ndarray, q: torch.Tensor, scale: torch.Tensor):
    want_q, want_s = I.quantize(x)
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert np.array_equal(scale.cpu().numpy(), want_s, equal_nan=True)


@pytest.mark.parametrize("M,K", [(1, 16), (3, 48), (5, 512), (2, 528), (7, 1024), (4, 1040), (3, 1536), (2, 1552),
                                 (1, 2048), (2, 2064), (5, 4096), (3, 4112), (2, 8192), (3, 8208), (1, 16384),
                                 (2, 16400), (1, 32768), (1025, 64), (300, 2048)])
def test_quant_codes_and_scales(hip, M, K):
    print(f"[case] quant {M} x {K}", flush=True)
    x = rows_of(np.random.default_rng(M * K), M, K)
    check_quant(x, *ops.quant_act_int8(bf16_tensor(x)))


def test_quant_ties_to_even_and_edges(hip):
    # a = 127 2^e: every multiple of 2^(e-1) is a half code or a whole one
    rows = []
    for e in (-90, -7, 0, 3, 100):
        halves = np.arange(-254, 255)
        v = np.concatenate([halves[np.abs(halves) < 256] * 2.0 ** (e - 1), [127.0 * 2.0 ** e]])
        rows.append(np.resize(F.bf16_round(v.astype(np.float32)), 512))
    # 254 x = (2h + 1) a at other pairs of significands, and the halves' neighbours
    rows.append(np.resize(np.array([254.0, 1.0, 3.0, 5.0, 127.0, 129.0, 253.0, 63.5], np.float32), 512))
    rows.append(np.resize(np.array([3.3895e38, -3.3895e38, 1e36, 1e30], np.float32), 512))     # the largest numbers
    rows.append(np.zeros(512, np.float32))
    rows.append(np.resize(np.array([2.0 ** -101, -(2.0 ** -108), 1e-40], np.float32), 512))    # below the least a
    rows.append(np.resize(np.array([2.0 ** -100, -(2.0 ** -101)], np.float32), 512))
    x = F.bf16_round(np.stack(rows).astype(np.float32))
    q, scale = ops.quant_act_int8(bf16_tensor(x))
    check_quant(x, q, scale)
    assert int(q.cpu()[7].abs().max()) == 0


def test_quant_rows_with_inf_or_nan_are_nan(hip):
    x = rows_of(np.random.default_rng(5), 6, 4096)
    x[1, 4095], x[2, 0], x[4, 1000] = np.inf, -np.inf, np.nan
    q, scale = ops.quant_act_int8(bf16_tensor(x))
    check_quant(x, q, scale)
    assert torch.isnan(scale).cpu().tolist() == [False, True, True, False, True, False]
    b = torch.ones((16, 4096), dtype=torch.int8, device="cuda")
    y = ops.int8_gemm(q, scale, b, torch.ones(16, device="cuda"))
    assert torch.isnan(y).all(1).cpu().tolist() == [False, True, True, False, True, False]


@pytest.mark.parametrize("M", [1, 9])
def test_quant_of_a_slice(hip, M):
    x = rows_of(np.random.default_rng(M), M, 2112)
    wide = bf16_tensor(x)
    check_quant(x[:, 576:], *ops.quant_act_int8(wide[:, 576:]))
    got = ops.quant_act_int8(wide[:1, 576:].as_strided((1, 1536), (0, 1)))
    check_quant(x[:1, 576:], *got)


def product_case(M, N, K, seed, residual):
    rng = np.random.default_rng(seed)
    a = rng.integers(-128, 128, (M, K)).astype(np.int8)
    b = rng.integers(-128, 128, (N, K)).astype(np.int8)
    sa = np.exp2(rng.uniform(-8, 2, M)).astype(np.float32)
    sb = np.exp2(rng.uniform(-12, -4, N)).astype(np.float32)
    r = F.bf16_round((rng.standard_normal((M, N)) * 50).astype(np.float32)) if residual else None
    return a, sa, b, sb, r


def on_gpu(a, sa, b, sb, r):
    return (*(torch.from_numpy(v).cuda() for v in (a, sa, b, sb)), None if r is None else bf16_tensor(r))


@pytest.mark.parametrize("M,N,K,residual", [
    (1, 8, 16, False), (1, 24576, 4096, False), (2, 1000, 1040, True), (5, 4096, 512, False), (16, 4096, 12288, True),
    (17, 72, 272, False), (31, 6144, 4096, False), (33, 200, 16, True), (48, 2048, 7168, False), (64, 640, 2064, True),
    (65, 264, 4096, False), (100, 7168, 2048, False), (127, 128, 128, True), (129, 136, 144, False),
    (300, 1000, 1552, True), (513, 4096, 512, False), (1000, 520, 4096, False), (1025, 2056, 272, True),
    (2000, 264, 128, False), (4099, 8, 48, False)])
def test_product_bits(hip, M, N, K, residual):
    print(f"[case] int8 product {M} x {N} x {K}", flush=True)
    case = product_case(M, N, K, M + N + K, residual)
    y = ops.int8_gemm(*on_gpu(*case))
    assert np.array_equal(bits(y), I.product(*case))


# A shape of each tile without and with K splits (tests/test_int8_plan.py checks that), most with K, N and M off the tile.
TILES = [(1, 8, 1392), (1, 1352, 7632), (1, 16, 5984), (1, 8, 6896), (5, 8, 16), (1, 680, 5808), (1, 16808, 272),
         (1, 2744, 12208), (21, 8, 32), (21, 4080, 7152), (19, 8, 4928), (17, 16712, 160), (33, 2912, 12272), (39, 8, 688),
         (3, 5192, 10688), (33, 8, 5680), (51, 24, 16), (2703, 8, 3216), (33, 8, 2544), (65, 8480, 16), (65, 2704, 5920),
         (2867, 8, 5664), (67, 17064, 16), (67, 5968, 8112), (3589, 2056, 16), (217, 21168, 16), (69, 10968, 1072),
         (563, 19600, 16), (1025, 4104, 4112), (300, 24584, 528)]


@pytest.mark.parametrize("M,N,K", TILES)
def test_product_bits_of_every_tile(hip, M, N, K):
    """Against whole numbers summed on the GPU in 64 bits (exact below 2^53), then rounded as the oracle rounds."""
    print(f"[case] int8 product {M} x {N} x {K}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a, b = (torch.randint(-128, 128, (n, K), generator=g, device="cuda", dtype=torch.int8) for n in (M, N))
    sa, sb = (torch.rand(n, generator=g, device="cuda") + 0.01 for n in (M, N))
    r = torch.randn((M, N), generator=g, device="cuda").to(torch.bfloat16) if M % 4 == 1 else None
    y = ops.int8_gemm(a, sa, b, sb, r)
    total = (a.double() @ b.double().t()).float()
    want = total * sa[:, None] * sb
    want = (want if r is None else want + r.float()).to(torch.bfloat16)
    assert torch.equal(y.view(torch.int16), want.view(torch.int16))


def test_product_largest_sums(hip):
    """K = 65536 of -128 * -128: 2^30, and 127 * -128 beside it."""
    K = 65536
    a = np.full((3, K), -128, np.int8)
    a[1], a[2, ::2] = 127, 127
    b = np.full((24, K), -128, np.int8)
    b[1], b[2, 1::2] = 127, 0
    sa, sb = np.array([1.0, 1e-3, 2e-5], np.float32), np.linspace(1e-4, 3, 24).astype(np.float32)
    y = ops.int8_gemm(*on_gpu(a, sa, b, sb, None))
    assert np.array_equal(bits(y), I.product(a, sa, b, sb))


def test_product_is_the_same_for_every_batch(hip):
    """A token's bits do not depend on the tokens around it, which choose tile and split."""
    a, sa, b, sb, _ = on_gpu(*product_case(700, 2048, 4096, 3, False))
    whole = ops.int8_gemm(a, sa, b, sb)
    for lo, n in ((0, 1), (3, 9), (40, 33), (5, 100), (100, 300)):
        part = ops.int8_gemm(a[lo:lo + n].contiguous(), sa[lo:lo + n].contiguous(), b, sb)
        assert torch.equal(part.view(torch.int16), whole[lo:lo + n].view(torch.int16)), (lo, n)


def test_product_in_place_on_the_residual(hip):
    case = product_case(20, 520, 4096, 8, True)
    a, sa, b, sb, r = on_gpu(*case)
    y = ops.int8_gemm(a, sa, b, sb, r, out=r)
    assert y.data_ptr() == r.data_ptr() and np.array_equal(bits(y), I.product(*case))


def test_outputs_and_workspaces_of_the_caller(hip):
    case = product_case(8, 4096, 12288, 9, False)
    t = on_gpu(*case)[:4]
    need = ops.int8_gemm_workspace_bytes(8, 4096, 12288)
    out = torch.full((9, 4096), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((need + 64,), 0x5a, dtype=torch.uint8, device="cuda")
    y = ops.int8_gemm(*t, out=out[:8], workspace=ws)
    assert np.array_equal(bits(y), I.product(*case))
    assert (out[8] == 7).all() and (ws[need:] == 0x5a).all()
    y = ops.int8_gemm(*t, workspace=torch.empty(4, dtype=torch.uint8, device="cuda"))
    assert np.array_equal(bits(y), I.product(*case))


def test_refusals(hip):
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    a, b = (torch.zeros((n, 256), dtype=torch.int8, device="cuda") for n in (4, 32))
    sa, sb = torch.ones(4, device="cuda"), torch.ones(32, device="cuda")
    with pytest.raises(TypeError):
        ops.quant_act_int8(x.float())
    with pytest.raises(ValueError):
        ops.quant_act_int8(x[:1].expand(4, 256))
    with pytest.raises(lib.FerretError):
        ops.quant_act_int8(x[:, :200].contiguous())
    with pytest.raises(lib.FerretError):
        ops.quant_act_int8(x, q=x.view(torch.int8).view(-1)[:1024].view(4, 256))   # over x
    with pytest.raises(TypeError):
        ops.int8_gemm(a.float(), sa, b, sb)
    with pytest.raises(ValueError):
        ops.int8_gemm(a, sa, b[:, :128].contiguous(), sb)
    with pytest.raises(ValueError):
        ops.int8_gemm(a, sa[:3], b, sb)
    with pytest.raises(ValueError):
        ops.int8_gemm(a, sa, b, sb, out=torch.empty((4, 24), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        ops.int8_gemm(a.t(), sa, b, sb)
    with pytest.raises(lib.FerretError):
        ops.int8_gemm(a, sa, b[:28].contiguous(), sb[:28].contiguous())     # N % 8
    with pytest.raises(lib.FerretError):
        ops.int8_gemm(a, sa, b, torch.ones(33, device="cuda")[1:])          # off its bound
    with pytest.raises(lib.FerretError):
        ops.int8_gemm(a, sa, b, sb, out=b.view(-1)[:256].view(torch.bfloat16).view(4, 32))


def test_another_stream_and_captured_replays(hip):
    """Quantizer and split product on a side stream, then captured: every replay has the eager bits."""
    rng = np.random.default_rng(11)
    b = torch.from_numpy(rng.integers(-128, 128, (4096, 12288)).astype(np.int8)).cuda()
    sb = torch.full((4096,), 1e-3, device="cuda")
    xs = [bf16_tensor(rows_of(rng, 8, 12288)) for _ in range(3)]
    x, r = xs[0].clone(), bf16_tensor(rows_of(rng, 8, 4096))
    eager = [ops.int8_gemm(*ops.quant_act_int8(v), b, sb, r) for v in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.int8_gemm(*ops.quant_act_int8(x), b, sb, r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, eager[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.int8_gemm(*ops.quant_act_int8(x), b, sb, r)
    for i in (1, 2, 0, 1):
        x.copy_(xs[i])
        y.fill_(-1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.int16), eager[i].view(torch.int16)), i


def test_native_and_python_paths_agree(hip, monkeypatch):
    case = on_gpu(*product_case(12, 4096, 4096, 21, True))
    x = bf16_tensor(rows_of(np.random.default_rng(2), 12, 4096))
    nat = lib.native()
    assert nat.quant_act_int8(x, None, None) is not None and nat.int8_gemm(*case, None, None) is not None
    here = [*ops.quant_act_int8(x), ops.int8_gemm(*case)]
    monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    there = [*ops.quant_act_int8(x), ops.int8_gemm(*case)]
    for u, v in zip(here, there):
        assert u.dtype == v.dtype and torch.equal(u.view(torch.uint8), v.view(torch.uint8))


def test_offsets_past_32_bits(hip):
    """Tokens and weights of more than 2^32 bytes: the last rows as they are alone."""
    print("[case] int8 far rows", flush=True)
    K, far = 32768, 140000
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.zeros((far, K), dtype=torch.bfloat16, device="cuda")
    x[-70:] = torch.randn((70, K), generator=g, device="cuda").to(torch.bfloat16)
    q, s = ops.quant_act_int8(x)
    few = x[-70:].clone()
    del x
    tq, ts = ops.quant_act_int8(few)
    check_quant(few.float().cpu().numpy(), tq, ts)
    assert torch.equal(q[-70:], tq) and torch.equal(s[-70:], ts) and not q[:-70].any()
    w, ws = ops.quant_act_int8(torch.randn((72, K), generator=g, device="cuda").to(torch.bfloat16))
    want = I.product(*(t.cpu().numpy() for t in (tq, ts, w, ws)))
    assert np.array_equal(bits(ops.int8_gemm(q, s, w, ws)[-70:]), want)
    for M in (1, 70):       # q as weights
        y = ops.int8_gemm(w[:M].contiguous(), ws[:M].contiguous(), q, s)
        assert np.array_equal(bits(y)[:, -70:], I.product(*(t.cpu().numpy() for t in (w[:M], ws[:M], tq, ts))))
        assert not y[:, :-70].any()
