"""GPU: the int8 operators and the attention over shared prefixes together, as a model's layer calls them: a prompt
that several samples continue, its keys once in the cache; by the native call path, the Python one, torch.ops and
a captured graph.

Every int8 product is checked for its bits from the codes that it was given, the attention against the formula in
64 bits over the keys that the cache holds.
"""
import numpy as np
import pytest
import torch

from ferret_amd import lib
from oracle import attention as A
from oracle import int8 as I
from tests.attention_helpers import i32, starts, visible

pytestmark = pytest.mark.gpu

HID, QL, H, PAGE, SCALE = 1024, 512, 8, 32, 192.0 ** -0.5


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


def _values(t):
    return t.float().cpu().numpy()


class Layer:
    """An attention layer with int8 projections, a scale per output channel: the quantizer's, on the weight's rows."""

    def __init__(self, ops, seed=0):
        self.ops, g = ops, torch.Generator(device="cuda").manual_seed(seed)

        def weight(n, k):
            return (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).to(torch.bfloat16)
        self.down, self.up, self.out = (ops.quant_act_int8(weight(n, k)) for n, k in
                                        ((QL + 576, HID), (H * 192, QL), (HID, H * 128)))
        self.wk = [weight(512, 128) for _ in range(H)]
        self.wv = [weight(128, 512) for _ in range(H)]
        self.wn, self.wq, self.wl = ((1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(torch.bfloat16)
                                     for n in (HID, QL, 512))
        self.products = []

    def product(self, x, weight, residual=None):
        q, s = self.ops.quant_act_int8(x)
        y = self.ops.int8_gemm(q, s, *weight, residual)
        self.products.append((x, q, s, weight, residual, y))
        return y

    def check_products(self):
        for x, q, s, (w, sw), residual, y in self.products:
            want_q, want_s = I.quantize(_values(x))
            assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s)
            want = I.product(q.cpu().numpy(), s.cpu().numpy(), w.cpu().numpy(), sw.cpu().numpy(),
                             None if residual is None else _values(residual))
            assert np.array_equal(y.view(torch.int16).cpu().numpy().view(np.uint16), want)
        self.products.clear()

    def queries(self, x, cache, table, lens, cu_q):
        """Norm, projections and the new tokens' rows of the cache; the absorbed queries."""
        ops = self.ops
        h, _ = ops.rms_norm(x, self.wn)
        down = self.product(h, self.down)
        c, _ = ops.rms_norm(down[:, :QL], self.wq)
        q = self.product(c, self.up).view(-1, H, 192)
        lat, _ = ops.rms_norm(down[:, QL:QL + 512], self.wl)
        ops.latent_cache_write(cache, lat, down[:, QL + 512:], table, lens, cu_q)
        ql = torch.stack([ops.linear_bf16(q[:, h, :128].contiguous(), self.wk[h]) for h in range(H)], 1)
        return ql, q[..., 128:]

    def finish(self, x, o):
        o = torch.cat([self.ops.linear_bf16(o[:, h].contiguous(), self.wv[h]) for h in range(H)], 1)
        return self.product(o, self.out, x)

    def prompt(self, x, cache, table, lens, cu_q):
        ql, qr = self.queries(x, cache, table, lens, cu_q)
        return self.finish(x, self.ops.latent_attention(ql, qr, cache, table, lens, cu_q, SCALE))

    def step(self, x, cache, prefix, own):
        """One step of samples: `prefix` is (table, lens, cu_prefix), `own` (table, lens, cu_q)."""
        ql, qr = self.queries(x, cache, *own)
        o, lse = self.ops.latent_attention_shared(ql, qr, cache, *prefix, *own, SCALE, return_lse=True)
        return self.finish(x, o), ql, qr, o, lse


PROMPTS, SAMPLES, STEPS = [70, 33], [3, 2], [[1, 1, 1, 1, 1], [1, 4, 1, 2, 1], [1, 1, 1, 1, 1]]


class Run:
    """The prompts in pages 0 to 4, each sample's own tokens in one page."""

    def __init__(self, ops, layer, e4m3):
        self.ops, self.layer = ops, layer
        self.cache = ops.LatentCache.empty(10, PAGE, torch.float8_e4m3fn if e4m3 else torch.bfloat16)
        self.table, self.lens = i32([3, 1, 0, 4, 2, -1]).view(2, 3), i32(PROMPTS)
        self.cu_prefix, self.own, self.have = i32([0, 3, 5]), i32([8, 5, 6, 9, 7]).view(5, 1), [0] * 5
        self.g = torch.Generator(device="cuda").manual_seed(5)
        layer.prompt(self.random(sum(PROMPTS)), self.cache, self.table, self.lens, i32(starts(PROMPTS)))

    def random(self, n):
        return torch.randn((n, HID), generator=self.g, device="cuda").to(torch.bfloat16)

    def step(self, new):
        self.have = [a + b for a, b in zip(self.have, new)]
        cu_q = i32(starts(new))
        cu_prefix = i32([0, sum(new[:SAMPLES[0]]), sum(new)])
        return self.layer.step(self.random(sum(new)), self.cache, (self.table, self.lens, cu_prefix),
                               (self.own, i32(self.have), cu_q))


@pytest.mark.parametrize("e4m3", [False, True])
def test_samples_of_prompts(ops, e4m3):
    print(f"[case] int8 block e4m3={e4m3}", flush=True)
    layer = Layer(ops)
    run = Run(ops, layer, e4m3)
    for new in STEPS:
        y, ql, qr, o, lse = run.step(new)
        torch.cuda.synchronize()
        layer.check_products()
        assert torch.isfinite(y.float()).all()
        groups = [0] * SAMPLES[0] + [1] * SAMPLES[1]
        t = 0
        for b, n in enumerate(new):
            p = groups[b]
            parts = [ops.latent_cache_read(run.cache, tab, i32([0, m]), m) for tab, m in
                     ((run.table[p:p + 1], PROMPTS[p]), (run.own[b:b + 1], run.have[b]))]
            lat, rot = (np.concatenate([_values(part[i]) for part in parts]) for i in (0, 1))
            k = np.concatenate([lat, rot], 1)
            see = np.concatenate([np.ones((n, PROMPTS[p]), dtype=bool), visible(n, run.have[b])], 1)
            for h in range(H):
                q = np.concatenate([_values(ql[t:t + n, h]), _values(qr[t:t + n, h])], 1)
                want, ref, spread, reach = A.attend(q, k, lat, SCALE, see)
                eo, el = A.bounds(want, ref, spread, reach, 576, len(k))
                assert (np.abs(_values(o[t:t + n, h]) - want) <= eo).all(), (b, h)
                assert (np.abs(lse[t:t + n, h].cpu().numpy() - ref) <= el).all(), (b, h)
            t += n


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
    print("[case] int8 block native path", flush=True)
    rec = _Recorder(lib.native())
    monkeypatch.setattr(lib, "native", lambda: rec)
    here = Run(ops, Layer(ops), True).step(STEPS[1])
    assert rec.took >= {"quant_act_int8", "int8_gemm", "latent_attention_shared"} and not rec.left
    monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    there = Run(ops, Layer(ops), True).step(STEPS[1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(here, there))


def test_torch_ops_and_a_compiled_step(ops):
    print("[case] int8 block torch.ops", flush=True)
    import ferret_amd.torch_ops  # noqa: F401
    T = torch.ops.ferret
    layer = Layer(ops)
    run = Run(ops, layer, True)
    _, ql, qr, o, lse = run.step(STEPS[0])
    x = run.random(5)
    tests = ("test_schema", "test_faketensor")
    q, s = T.quant_act_int8(x)
    torch.library.opcheck(T.quant_act_int8.default, (x,), test_utils=tests)
    torch.library.opcheck(T.int8_gemm.default, (q, s, *layer.down), test_utils=tests)
    torch.library.opcheck(T.int8_gemm.default, (q, s, layer.down[0][:HID], layer.down[1][:HID], x), test_utils=tests)
    args = (ql, qr, run.cache.data, run.cache.scales, run.table, run.lens, run.cu_prefix, run.own, i32(run.have),
            i32(range(6)), SCALE)
    torch.library.opcheck(T.latent_attention_shared.default, args, test_utils=tests)

    def step(x, ql):
        a = T.int8_gemm(*T.quant_act_int8(x), *layer.down)
        return a, T.latent_attention_shared(ql, *args[1:])
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(x, ql)
    assert torch.equal(got[0], ops.int8_gemm(*ops.quant_act_int8(x), *layer.down))
    assert torch.equal(got[1][0], o) and torch.equal(got[1][1], lse)


def test_a_step_captured_and_replayed(ops):
    """A whole step of the samples in a graph, replayed as their own parts grow, against the eager step on another cache."""
    print("[case] int8 block graph", flush=True)
    layer = Layer(ops)
    one, two = Run(ops, layer, True), Run(ops, layer, True)
    x, lens, cu = torch.zeros((5, HID), dtype=torch.bfloat16, device="cuda"), i32([1] * 5), i32(range(6))

    def step(run):
        return layer.step(x, run.cache, (run.table, run.lens, run.cu_prefix), (run.own, lens, cu))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(one)
    for k in range(20):
        x.copy_(two.random(5))
        lens.fill_(k + 1)
        g.replay()
        want = step(two)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
        assert torch.equal(one.cache.data, two.cache.data) and torch.equal(one.cache.scales, two.cache.scales), k


def test_two_graphs_on_one_workspace(ops):
    """Graphs of other products and batches, captured on the same workspaces and replayed in turn."""
    print("[case] int8 block shared workspaces", flush=True)
    g = torch.Generator(device="cuda").manual_seed(8)
    shapes = [(3, 64, 32768), (100, 512, 16384)]
    need = max(ops.int8_gemm_workspace_bytes(*s) for s in shapes)
    assert min(ops.int8_gemm_workspace_bytes(*s) for s in shapes) > 0
    layer = Layer(ops)
    runs = [Run(ops, layer, e4m3) for e4m3 in (True, False)]
    states = [run.step(new) for run, new in zip(runs, STEPS[:2])]
    attention = ops.latent_attention_shared_workspace_bytes(2, 5, 9, H)
    ws, ws2 = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (need, attention))
    calls, want = [], []
    for (M, N, K), run, (_, ql, qr, _, _), new in zip(shapes, runs, states, STEPS):
        a, b = (ops.quant_act_int8(torch.randn((n, K), generator=g, device="cuda").to(torch.bfloat16)) for n in (M, N))
        index = (run.table, run.lens, i32([0, sum(new[:SAMPLES[0]]), sum(new)]), run.own, i32(run.have), i32(starts(new)))

        def call(a=a, b=b, ql=ql, qr=qr, cache=run.cache, index=index):
            return (ops.int8_gemm(*a, *b, workspace=ws),
                    ops.latent_attention_shared(ql, qr, cache, *index, SCALE, workspace=ws2))
        want.append(tuple(t.clone() for t in call()))
        calls.append(call)
    graphs = [torch.cuda.CUDAGraph() for _ in calls]
    out = []
    for graph, call in zip(graphs, calls):
        with torch.cuda.graph(graph):
            out.append(call())
    for i in (0, 1, 1, 0, 1, 0):
        for t in out[i]:
            t.fill_(7)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out[i], want[i])), i
        calls[1 - i]()
