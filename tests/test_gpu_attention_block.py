"""GPU: the operators together, as a model's attention layer calls them: norm into the FP8
projections, the cache's write, and both forms of the attention over it; by torch.ops, by the
native call path and by the Python one, and captured into a graph.

The absorbed and the expanded form of one layer are the same function of the hidden
states up to roundings: the test states that bound from the roundings in between.
"""
import numpy as np
import pytest
import torch

from ferret_amd import lib
from tests.attention_helpers import i32, starts

pytestmark = pytest.mark.gpu

HID, QL, H, SCALE = 1024, 512, 8, 192.0 ** -0.5


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


class Layer:
    """One attention layer's weights at a small hidden size: FP8 projections, bf16 key-value expansion."""

    def __init__(self, seed=0):
        from ferret_amd import workloads as W
        g = torch.Generator(device="cuda").manual_seed(seed)

        def w(n, k):
            return W.quant_weight_128x128(torch.randn((n, k), generator=g, device="cuda") * k ** -0.5)
        self.down, self.up = w(QL + 512 + 128, HID), w(H * 256, QL)      # (64 rotary, 64 unused), (128 + 64, 64 unused)
        self.kvb = (torch.randn((H * 256, 512), generator=g, device="cuda") * 512 ** -0.5).to(torch.bfloat16)
        self.wn, self.wq, self.wk = ((1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(torch.bfloat16)
                                     for n in (HID, QL, 512))

    def project(self, ops, x, residual, cache, table, lens, cu_q):
        q8, s8, residual = ops.rms_norm_e4m3(x, self.wn, residual)
        down = ops.fp8_gemm_blockscale(q8, s8, *self.down)
        q8, s8, _ = ops.rms_norm_e4m3(down[:, :QL], self.wq)
        q = ops.fp8_gemm_blockscale(q8, s8, *self.up).view(-1, H, 256)
        lat, _ = ops.rms_norm(down[:, QL:QL + 512], self.wk)
        ops.latent_cache_write(cache, lat, down[:, QL + 512:QL + 576], table, lens, cu_q)
        return q[..., :128], q[..., 128:192], residual

    def absorbed(self, ops, qn, qr, cache, table, lens, cu_q):
        wk, wv = self.kvb.view(H, 256, 512).split(128, 1)
        ql = torch.stack([qn[:, h].float() @ wk[h].float() for h in range(H)], 1).to(torch.bfloat16)
        o = ops.latent_attention(ql, qr, cache, table, lens, cu_q, SCALE)
        return torch.stack([o[:, h].float() @ wv[h].float().t() for h in range(H)], 1)

    def expanded(self, ops, qn, qr, cache, table, cu_k, total, cu_q):
        lat, rot = ops.latent_cache_read(cache, table, cu_k, total)
        kv = ops.linear_bf16(lat, self.kvb).view(total, H, 256)
        return ops.latent_attention_expanded(qn, qr, kv[..., :128], rot, kv[..., 128:], cu_q, cu_k, SCALE)


def _table(lens, page):
    per = [-(-n // page) for n in lens]
    t = torch.zeros((len(lens), max(per)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        t[b, :n] = torch.arange(at, at + n).flip(0)
        at += n
    return t, at


@pytest.mark.parametrize("e4m3", [False, True])
def test_prompt_then_tokens(ops, e4m3):
    """Two prompts of a batch, then three decode steps; every step in both forms."""
    print(f"[case] attention block e4m3={e4m3}", flush=True)
    layer, prompt, page = Layer(), [70, 33], 32
    table, pages = _table([n + 3 for n in prompt], page)
    cache = ops.LatentCache.empty(pages, page, torch.float8_e4m3fn if e4m3 else torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(5)
    for step in range(4):
        new = prompt if step == 0 else [1, 1]
        lens = [n + step for n in prompt]
        x, r = (torch.randn((sum(new), HID), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        cu_q, cu_k, dlens = i32(starts(new)), i32(starts(lens)), i32(lens)
        qn, qr, r2 = layer.project(ops, x, r, cache, table, dlens, cu_q)
        a = layer.absorbed(ops, qn, qr, cache, table, dlens, cu_q)
        e = layer.expanded(ops, qn, qr, cache, table, cu_k, sum(lens), cu_q).float()
        torch.cuda.synchronize()
        assert torch.equal(r2, (x.float() + r.float()).to(torch.bfloat16))
        # Between the two: the key projection's product rounded on the query's side or on the
        # key's (2^-8 of each score's sum of magnitudes at most: about 0.03 for scores of
        # unit variance over 128 terms, a relative 0.03 on the softmax terms), the values'
        # projection before or after the sum, and both outputs' roundings.  Over a row of 128
        # columns these average far below that: 0.03 of the row's norm bounds it.
        off = (a - e).norm(dim=-1) / e.norm(dim=-1)
        assert off.max() < 0.03, (step, float(off.max()))


def _calls(ops, layer):
    cache = ops.LatentCache.empty(12, 16, torch.float8_e4m3fn)
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    g = torch.Generator(device="cuda").manual_seed(6)
    x, r = (torch.randn((50, HID), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    lens, cu = i32([60, 30]), i32([0, 40, 50])
    y, r1 = ops.rms_norm(x, layer.wn, r)
    q8, s8, r2 = ops.rms_norm_e4m3(x, layer.wn, r)
    qn, qr, _ = layer.project(ops, x, r, cache, table, lens, cu)
    lat, rot = ops.latent_cache_read(cache, table, i32([0, 60, 90]), 90)
    ql = torch.randn((50, H, 512), generator=g, device="cuda").to(torch.bfloat16)
    o, lse = ops.latent_attention(ql, qr, cache, table, lens, cu, SCALE, return_lse=True)
    kv = ops.linear_bf16(lat, layer.kvb).view(90, H, 256)
    o2, lse2 = ops.latent_attention_expanded(qn, qr, kv[..., :128], rot, kv[..., 128:], cu, i32([0, 60, 90]), SCALE,
                                             causal=False, return_lse=True)
    return [y, r1, q8, s8, r2, cache.data, cache.scales, lat, rot, o, lse, o2, lse2]


class _Recorder:
    def __init__(self, nat):
        self.nat, self.took, self.left = nat, set(), set()

    def __getattr__(self, name):
        def call(*args):
            r = getattr(self.nat, name)(*args)
            (self.left if r is None else self.took).add(name)
            return r
        return call


def test_the_native_path_gives_the_bits_of_the_python_path(ops, monkeypatch):
    print("[case] attention block native path", flush=True)
    layer = Layer()
    rec = _Recorder(lib.native())
    monkeypatch.setattr(lib, "native", lambda: rec)
    here = _calls(ops, layer)
    assert rec.took >= {"rms_norm", "rms_norm_e4m3", "latent_cache_write", "latent_cache_read", "latent_attention",
                        "latent_attention_expanded"} and not rec.left
    monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    there = _calls(ops, layer)
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(here, there)):
        assert a.shape == b.shape and a.dtype == b.dtype
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), i


def test_torch_ops(ops):
    """opcheck of the schemas (the cache's mutation among them) and fakes, and a compiled layer step."""
    print("[case] attention block torch.ops", flush=True)
    import ferret_amd.torch_ops  # noqa: F401
    T = torch.ops.ferret
    layer = Layer()
    g = torch.Generator(device="cuda").manual_seed(7)
    x, r = (torch.randn((6, HID), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(T.rms_norm.default, (x, layer.wn), test_utils=tests)
    torch.library.opcheck(T.add_rms_norm.default, (x, r, layer.wn), test_utils=tests)
    cache = ops.LatentCache.empty(4, 16, torch.float8_e4m3fn)
    table, lens, cu = i32([0, 1, 2, 3]).view(2, 2), i32([20, 30]), i32([0, 2, 6])
    lat = torch.randn((6, 512), generator=g, device="cuda").to(torch.bfloat16)
    rot, qr = (torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in ((6, 64), (6, H, 64)))
    ql = torch.randn((6, H, 512), generator=g, device="cuda").to(torch.bfloat16)
    torch.library.opcheck(T.latent_cache_write.default, (cache.data, cache.scales, lat, rot, table, lens, cu),
                          test_utils=tests)
    torch.library.opcheck(T.latent_cache_read.default, (cache.data, cache.scales, table, i32([0, 20, 50]), 50),
                          test_utils=tests)
    torch.library.opcheck(T.latent_attention.default, (ql, qr, cache.data, cache.scales, table, lens, cu, SCALE),
                          test_utils=tests)
    kv = torch.randn((50, H, 256), generator=g, device="cuda").to(torch.bfloat16)
    kr = torch.randn((50, 64), generator=g, device="cuda").to(torch.bfloat16)
    torch.library.opcheck(T.latent_attention_expanded.default,
                          (ql[..., :128], qr, kv[..., :128], kr, kv[..., 128:], cu, i32([0, 20, 50]), SCALE),
                          test_utils=tests)

    def step(x, r, data, scales):
        q8, s8, r = T.add_rms_norm_e4m3(x, r, layer.wn)
        down = T.fp8_gemm_blockscale(q8, s8, *layer.down)
        T.latent_cache_write(data, scales, T.rms_norm(down[:, QL:QL + 512], layer.wk), down[:, QL + 512:QL + 576], table,
                             lens, cu)
        return T.latent_attention(ql, qr, data, scales, table, lens, cu, SCALE)[0], r

    one, two = (ops.LatentCache.empty(4, 16, torch.float8_e4m3fn) for _ in range(2))
    want = step(x, r, one.data, one.scales)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(x, r, two.data, two.scales)
    torch.cuda.synchronize()
    assert torch.equal(one.data, two.data) and torch.equal(one.scales, two.scales)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_step_captured_and_replayed(ops):
    """A whole decode step in a graph, replayed over growing lengths, against the eager step on a cache of its own."""
    print("[case] attention block graph", flush=True)
    layer, B = Layer(), 3
    table, pages = _table([64] * B, 16)
    one, two = (ops.LatentCache.empty(pages, 16, torch.float8_e4m3fn) for _ in range(2))
    x, r = (torch.zeros((B, HID), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lens, cu = i32([1] * B), i32(range(B + 1))

    def step(cache):
        qn, qr, res = layer.project(ops, x, r, cache, table, lens, cu)
        ql = torch.cat([qn, qn, qn, qn], -1)
        return ops.latent_attention(ql, qr, cache, table, lens, cu, SCALE), res
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(one)
    rng = np.random.default_rng(1)
    for k in range(20):
        x.copy_(torch.from_numpy(rng.standard_normal((B, HID))).cuda())
        r.copy_(torch.from_numpy(rng.standard_normal((B, HID))).cuda())
        lens.fill_(k + 1)
        g.replay()
        want = step(two)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k
        assert torch.equal(one.data, two.data) and torch.equal(one.scales, two.scales), k
