"""GPU: int8 products whose K is split, bit for bit against the oracle: workspaces of the caller, of the allocator and of
captured calls.  Every test asks that its shapes do have a workspace."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ferret_amd import lib, ops
from oracle import int8 as I
from tests.test_gpu_int8 import bf16_tensor, bits, on_gpu, product_case, rows_of

pytestmark = pytest.mark.gpu

# the kernel for few tokens, then those for more
SHAPES = [(1, 1352, 7632), (8, 1000, 12288), (20, 520, 4096), (33, 2048, 4096), (70, 2704, 5920), (100, 1000, 4096)]


def need_of(M, N, K):
    need = ops.int8_gemm_workspace_bytes(M, N, K)
    assert need > 0, "a shape that splits K no longer: take another"
    return need


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_workspace_of_the_caller(hip, M, N, K):
    """Garbage in it does not reach the result, nothing is written past it or past the output; a smaller one is not
    taken."""
    print(f"[case] int8 split {M} x {N} x {K}", flush=True)
    need = need_of(M, N, K)
    case = product_case(M, N, K, M + N, True)
    a, sa, b, sb, r = on_gpu(*case)
    want = I.product(*case)
    ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    out = torch.full((M + 1, N), 7.0, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):
        y = ops.int8_gemm(a, sa, b, sb, r, out=out[:M], workspace=ws[:need])
        assert y.data_ptr() == out.data_ptr() and np.array_equal(bits(y), want)
    assert (ws[:need] != 0x5a).any() and (ws[need:] == 0x5a).all() and (out[M] == 7).all()
    few = torch.full((need - 16,), 0x5a, dtype=torch.uint8, device="cuda")
    assert np.array_equal(bits(ops.int8_gemm(a, sa, b, sb, r, workspace=few)), want) and (few == 0x5a).all()
    y = ops.int8_gemm(a, sa, b, sb, r, out=r, workspace=ws)
    assert y.data_ptr() == r.data_ptr() and np.array_equal(bits(y), want)


def test_refusals(hip):
    M, N, K = 20, 520, 4096
    need = need_of(M, N, K)
    a, sa, b, sb, r = on_gpu(*product_case(M, N, K, 1, True))
    with pytest.raises(lib.FerretError):
        ops.int8_gemm(a, sa, b, sb, workspace=torch.empty(need + 16, dtype=torch.uint8, device="cuda")[8:need + 8])
    with pytest.raises(lib.FerretError):
        ops.int8_gemm(a, sa, b, sb, workspace=b.view(torch.uint8).view(-1)[:need])
    with pytest.raises(ValueError):
        ops.int8_gemm(a, sa, b, sb, workspace=torch.empty(need, dtype=torch.uint8))
    with pytest.raises(ValueError):
        ops.int8_gemm(a, sa, b, sb, workspace=torch.empty((need, 2), dtype=torch.uint8, device="cuda")[:, 0])


@pytest.mark.parametrize("M,N,K", [(20, 520, 4096), (70, 2704, 5920)])
def test_captured_replays(hip, M, N, K):
    """Quantizer and split product with the residual, captured: replays among eager calls of other sizes, each with the
    eager bits; two graphs with a workspace each."""
    print(f"[case] int8 split captured {M} x {N} x {K}", flush=True)
    need = need_of(M, N, K)
    rng = np.random.default_rng(M)
    b = torch.from_numpy(rng.integers(-128, 128, (N, K)).astype(np.int8)).cuda()
    sb = torch.full((N,), 1e-3, device="cuda")
    xs = [bf16_tensor(rows_of(rng, M, K)) for _ in range(3)]
    r = bf16_tensor(rows_of(rng, M, N))
    eager = [ops.int8_gemm(*ops.quant_act_int8(v), b, sb, r) for v in xs]
    assert np.array_equal(bits(eager[1]), I.product(*(t.cpu().numpy() for t in (*ops.quant_act_int8(xs[1]), b, sb)),
                                                    r.float().cpu().numpy()))
    graphs = []
    for _ in range(2):
        x, ws = xs[0].clone(), torch.empty(need, dtype=torch.uint8, device="cuda")
        ops.int8_gemm(*ops.quant_act_int8(x), b, sb, r, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.int8_gemm(*ops.quant_act_int8(x), b, sb, r, workspace=ws)
        graphs.append((g, x, y, ws))
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in (1, 2, 0, 1):
        for k, (g, x, y, ws) in enumerate(graphs):
            x.copy_(xs[(i + k) % 3])
            y.fill_(-1)
        torch.cuda.synchronize()
        for s, (g, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        ops.int8_gemm(*ops.quant_act_int8(xs[i][:5]), b, sb, r[:5])
        torch.cuda.synchronize()
        for k, (_, _, y, _) in enumerate(graphs):
            assert torch.equal(y.view(torch.int16), eager[(i + k) % 3].view(torch.int16)), (i, k)


def test_two_streams(hip):
    """Split products in flight on two streams, their workspaces from the allocator."""
    cases = [on_gpu(*product_case(*s, 5, True)) for s in ((33, 2048, 4096), (100, 1000, 4096))]
    for (a, _, b, *_) in cases:
        need_of(a.shape[0], b.shape[0], a.shape[1])
    want = [ops.int8_gemm(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.int8_gemm(*c))
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(y.view(torch.int16), w.view(torch.int16)) for y in ys)


def test_native_and_python_paths_agree(hip, monkeypatch):
    M, N, K = 33, 2048, 4096
    need = need_of(M, N, K)
    case = on_gpu(*product_case(M, N, K, 21, True))
    assert lib.native().int8_gemm(*case, None, None) is not None
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    here = [ops.int8_gemm(*case), ops.int8_gemm(*case, workspace=ws)]
    monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    there = [ops.int8_gemm(*case), ops.int8_gemm(*case, workspace=ws)]
    for u in (*here, *there):
        assert torch.equal(u.view(torch.int16), here[0].view(torch.int16))
