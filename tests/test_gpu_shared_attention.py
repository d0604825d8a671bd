"""GPU: latent attention over shared prefixes against the formula in 64 bits (oracle.attention), with
bounds that count every rounding (oracle.attention.bounds)."""
import numpy as np
import pytest
import torch

from ferret_amd import lib
from oracle import attention as A
from tests.attention_helpers import SCALE, Batch, assert_near, bf16_tensor, bf16_values, i32, starts, visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


class Shared:
    """Prefixes and sequences of one cache: `groups` gives (prefix length, [(own keys, new tokens), ...]) in order,
    prefix length None for sequences behind all of the prefixes, or before them."""

    def __init__(self, groups, H, page, e4m3, seed, poison=False, std=1.0):
        self.groups, self.H, self.page = groups, H, page
        self.prefix = [p for p, _ in groups if p is not None]
        self.own = [s for _, members in groups for s in members]
        self.G, lens = len(self.prefix), [k for k, _ in self.own]
        self.new = [n for _, n in self.own]
        self.batch = Batch(self.prefix + lens, page, e4m3, seed, poison=poison)
        self.tokens = [sum(n for _, n in members) for p, members in groups]
        first = next((i for i, (p, _) in enumerate(groups) if p is not None), 0)
        self.before = sum(self.tokens[:first])
        at = starts([t for t, (p, _) in zip(self.tokens, groups) if p is not None])
        self.cu_prefix = [self.before + x for x in at]
        rng = np.random.default_rng(seed + 1)
        T = max(1, sum(self.new))
        self.ql, self.qr = bf16_values(rng, T, H, 512, std=std), bf16_values(rng, T, H, 64, std=std)

    def index(self):
        table = torch.from_numpy(self.batch.table).cuda()
        return dict(prefix_table=table[:self.G].contiguous(), prefix_lens=i32(self.prefix), cu_prefix=i32(self.cu_prefix),
                    page_table=table[self.G:].contiguous(), lens=i32([k for k, _ in self.own]),
                    cu_q=i32(starts(self.new)))

    def call(self, ops, **more):
        kw = dict(scale=SCALE, return_lse=True)
        kw.update(self.index())
        kw.update(more)
        return ops.latent_attention_shared(bf16_tensor(self.ql), bf16_tensor(self.qr), self.batch.cache, **kw)

    def check(self, out, lse, causal=True, scale=SCALE):
        out, lse = out.float().cpu().numpy(), lse.cpu().numpy()
        t, line, g, worst = 0, self.G, 0, 0.0
        for p, members in self.groups:
            for own, n in members:
                lat, rot, see = self.batch.lat[line], self.batch.rot[line], visible(n, own, causal)
                if p is not None:
                    lat, rot = np.concatenate([self.batch.lat[g], lat]), np.concatenate([self.batch.rot[g], rot])
                    see = np.concatenate([np.ones((n, p), dtype=bool), see], 1)
                k = np.concatenate([lat, rot], 1)
                for h in range(self.H):
                    q = np.concatenate([self.ql[t:t + n, h], self.qr[t:t + n, h]], 1)
                    o, ref, spread, reach = A.attend(q, k, lat, scale, see)
                    eo, el = A.bounds(o, ref, spread, reach, 576, len(k))
                    worst = max(worst, assert_near(out[t:t + n, h], o, eo, f"prefix {p} own {own} head {h}"))
                    assert_near(lse[t:t + n, h], ref, el, f"lse prefix {p} own {own} head {h}")
                t, line = t + n, line + 1
            g += p is not None
        return worst

    def wide(self):
        """The index with a prefix table wide enough that prefixes get a pass of their own, or None where the rows
        do not: entries past the lengths are no pages."""
        T, B = sum(self.new), len(self.own)
        rows = T * self.H // B
        saved = min(B, T) * (10 if rows <= 16 else 17) - self.G * -(-(-(-T * self.H // self.G)) // 64) * 30
        if rows > 32 or saved <= 0:
            return None
        kw = self.index()
        steps = -(-6400 // saved)
        columns = -(-steps * 64 // self.page) + 1
        table = torch.full((self.G, max(columns, kw["prefix_table"].shape[1])), -1, dtype=torch.int32, device="cuda")
        table[:, :kw["prefix_table"].shape[1]] = kw["prefix_table"]
        return dict(kw, prefix_table=table)

    def run(self, ops, causal=True):
        out, lse = self.call(ops, causal=causal)
        torch.cuda.synchronize()
        print(f"    worst {self.check(out, lse, causal):.3f} of the bound", flush=True)
        wide = self.wide()
        if wide is not None:
            two = self.call(ops, causal=causal, **wide)
            torch.cuda.synchronize()
            print(f"    worst {self.check(*two, causal):.3f} of the bound, prefixes in a pass of their own", flush=True)
        return out, lse


ONE = [(1, 1), (15, 1), (64, 1), (65, 1), (130, 1)]


@pytest.mark.parametrize("H", [1, 3, 16, 17, 40, 64, 128])
@pytest.mark.parametrize("e4m3", [False, True])
def test_one_token_per_sequence(ops, H, e4m3):
    print(f"[case] shared decode H={H} e4m3={e4m3}", flush=True)
    Shared([(700, ONE)], H, 48, e4m3, H).run(ops)


@pytest.mark.parametrize("prefix", [1, 15, 16, 63, 64, 65, 127, 129])
@pytest.mark.parametrize("e4m3", [False, True])
def test_short_prefixes(ops, prefix, e4m3):
    print(f"[case] shared prefix of {prefix} e4m3={e4m3}", flush=True)
    Shared([(prefix, [(3, 1), (70, 2)])], 16, 16, e4m3, prefix).run(ops)


@pytest.mark.parametrize("H", [2, 16, 100])
@pytest.mark.parametrize("e4m3", [False, True])
def test_several_prefixes(ops, H, e4m3):
    """Prefixes of many lengths, an empty one and one without sequences; one token, several, chunks."""
    print(f"[case] shared groups H={H} e4m3={e4m3}", flush=True)
    Shared([(1000, [(5, 1), (40, 3), (200, 33)]), (0, [(17, 1), (64, 64)]), (300, []), (65, [(1, 1)])], H, 32, e4m3,
           5).run(ops)


@pytest.mark.parametrize("e4m3", [False, True])
def test_tokens_outside_the_prefixes(ops, e4m3):
    """Sequences before and behind all prefixes see their own keys only."""
    print(f"[case] shared with others e4m3={e4m3}", flush=True)
    Shared([(None, [(90, 2), (7, 1)]), (500, [(30, 1), (2, 2)]), (64, [(100, 5)]), (None, [(65, 1), (130, 3)])], 16, 16,
           e4m3, 6).run(ops)


@pytest.mark.parametrize("e4m3", [False, True])
def test_rows_without_own_keys_or_any(ops, e4m3):
    """A token with no own key sees the prefix alone; without a prefix it gets zeros and -inf."""
    print(f"[case] shared empty rows e4m3={e4m3}", flush=True)
    s = Shared([(130, [(0, 1), (1, 3), (40, 1)]), (0, [(0, 2), (3, 5)])], 16, 16, e4m3, 7)
    out, lse = s.run(ops)
    assert (out[5:7] == 0).all() and torch.isneginf(lse[5:7]).all()
    assert (out[7:9] == 0).all() and torch.isfinite(lse[9:]).all()


def test_all_own_keys_visible(ops):
    print("[case] shared non-causal", flush=True)
    Shared([(200, [(70, 3), (5, 5)]), (10, [(129, 1)])], 8, 32, True, 4).run(ops, causal=False)


@pytest.mark.parametrize("H,prefix,own", [(16, 9000, [(40, 1)]), (128, 5000, [(2500, 1), (1, 1)]), (16, 100, [(7000, 1)]),
                                          (2, 4000, [(3000, 1), (3, 1), (64, 1)])])
@pytest.mark.parametrize("e4m3", [False, True])
def test_long_parts_are_cut_and_joined(ops, H, prefix, own, e4m3):
    print(f"[case] shared long H={H} prefix={prefix} own={own} e4m3={e4m3}", flush=True)
    Shared([(prefix, own)], H, 64, e4m3, 3).run(ops)


def test_more_rows_than_work_groups(ops):
    """Whole tiles, several to a work-group, in both passes; most of the rows checked by a few sequences."""
    print("[case] shared 400 sequences", flush=True)
    Shared([(130, [(1 + 7 * i % 90, 1) for i in range(300)]), (70, [(3, 1) for _ in range(100)])], 16, 16, True, 9).run(ops)


def test_many_prefixes(ops):
    print("[case] shared 300 prefixes", flush=True)
    Shared([(7 * i % 100, [(1 + i % 20, 1)] * (i % 3)) for i in range(300)], 4, 16, False, 10).run(ops)


def test_large_scores(ops):
    print("[case] shared large scores", flush=True)
    for e4m3 in (False, True):
        Shared([(400, [(300, 2), (20, 1)])], 16, 64, e4m3, 8, std=8.0).run(ops)


@pytest.mark.parametrize("H,tokens", [(16, 1), (64, 1), (16, 9)])
def test_latents_past_448(ops, H, tokens):
    """Exponent bytes above 127 in some rows and blocks of 128 latents, in prefix and own keys."""
    print(f"[case] shared large latents H={H} tokens={tokens}", flush=True)
    s = Shared([(200, [(90, tokens), (40, tokens)])], H, 16, True, 20)
    scales = s.batch.cache.scales.view(-1, 4)
    rng = np.random.default_rng(21)
    byte = scales.cpu().numpy()
    for line, slots in enumerate(s.batch.slots):
        pick = rng.random((len(slots), 4)) < 0.1
        more = rng.integers(1, 7, (len(slots), 4)) * pick
        byte[slots] += more.astype(np.uint8)
        s.batch.lat[line] = s.batch.lat[line] * np.repeat(np.exp2(more), 128, axis=1)
    assert (byte > 127).any()
    scales.copy_(torch.from_numpy(byte))
    s.ql = s.ql * 2.0 ** -9
    s.run(ops)


@pytest.mark.parametrize("e4m3", [False, True])
def test_unseen_rows_do_not_reach(ops, e4m3):
    """NaN in every slot that no key has, pages' ends among them."""
    print(f"[case] shared poisoned slots e4m3={e4m3}", flush=True)
    Shared([(75, [(20, 1), (33, 7)]), (130, [(1, 1)])], 16, 48, e4m3, 12, poison=True).run(ops)


def test_nan_in_one_prefix_stays_with_its_tokens(ops):
    print("[case] shared NaN in a prefix", flush=True)
    s = Shared([(100, [(9, 1), (70, 2)]), (100, [(30, 2)])], 16, 16, False, 13)
    want, _ = s.call(ops)
    row = s.batch.slots_of(0, 100)[41]
    s.batch.cache.data.view(-1, 576)[row, 5] = float("nan")
    got, _ = s.call(ops)
    assert torch.isnan(got[:3]).all() and torch.equal(got[3:], want[3:])


def test_entries_that_are_no_page(ops):
    """A prefix page and an own page that name nothing: their keys are left out."""
    print("[case] shared missing pages", flush=True)
    s = Shared([(96, [(48, 1), (20, 2)])], 16, 16, True, 14)
    kw = s.index()
    kw["prefix_table"][0, 2], kw["page_table"][0, 1] = -1, s.batch.pages
    out, lse = s.call(ops, **kw)
    for line, page in ((0, 2), (1, 1)):
        keep = np.ones(s.batch.lens[line], dtype=bool)
        keep[16 * page:16 * page + 16] = False
        s.batch.lat[line], s.batch.rot[line] = s.batch.lat[line][keep], s.batch.rot[line][keep]
    s.groups = [(80, [(32, 1), (20, 2)])]
    s.check(out, lse)


def test_lengths_past_the_tables_and_below_zero(ops):
    """Lengths are cut to the tables, negative ones are none."""
    print("[case] shared lengths out of range", flush=True)
    s = Shared([(64, [(32, 1)]), (32, [(16, 1)])], 16, 16, False, 15)
    kw = s.index()
    columns = kw["prefix_table"].shape[1]
    assert columns == 4
    want, _ = s.call(ops)
    kw["prefix_lens"] = i32([1 << 30, 32])
    kw["lens"] = i32([32, -5])
    out, lse = s.call(ops, **kw)
    assert torch.equal(out[0], want[0])
    alone = Shared([(64, [(32, 1)]), (32, [(0, 1)])], 16, 16, False, 15)
    alone.batch, alone.ql, alone.qr = s.batch, s.ql, s.qr
    s.batch.lat[3], s.batch.rot[3] = s.batch.lat[3][:0], s.batch.rot[3][:0]
    alone.check(out, lse)


def test_is_the_attention_of_the_joined_table(ops):
    """A prefix of whole pages before a sequence's own is latent_attention over the joined table, to rounding."""
    print("[case] shared against joined tables", flush=True)
    s = Shared([(128, [(40, 1), (100, 3)])], 16, 32, True, 16)
    kw = s.index()
    out, lse = s.run(ops)
    table = torch.cat([kw["prefix_table"][:, :4].expand(2, -1), kw["page_table"]], 1).contiguous()
    ref, ref_lse = ops.latent_attention(bf16_tensor(s.ql), bf16_tensor(s.qr), s.batch.cache, table, kw["lens"] + 128,
                                        kw["cu_q"], SCALE, return_lse=True)
    s.check(ref, ref_lse)
    assert (out.float() - ref.float()).abs().max() < 2 ** -6 * ref.float().abs().max()


@pytest.mark.parametrize("e4m3", [False, True])
def test_strides_places_and_rows_behind(ops, e4m3):
    """Queries head by head and inside a wider projection, outputs of the caller, rows behind the last sequence
    left alone, the output in place on packed queries: the bits of the plain call."""
    print(f"[case] shared strides e4m3={e4m3}", flush=True)
    s = Shared([(300, [(30, 1), (65, 4)])], 16, 16, e4m3, 17)
    want, want_lse = s.run(ops)
    ql, qr, kw = bf16_tensor(s.ql), bf16_tensor(s.qr), s.index()
    heads = ql.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((5, 16, 192), dtype=torch.bfloat16, device="cuda")
    wide[..., 128:] = qr
    out, lse = ops.latent_attention_shared(heads, wide[..., 128:], s.batch.cache, **kw, scale=SCALE, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    more_l, more_r = torch.cat([ql, ql[:3]]), torch.cat([qr, qr[:3]])
    out = torch.full((8, 16, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.latent_attention_shared(more_l, more_r, s.batch.cache, **kw, scale=SCALE, out=out)
    assert torch.equal(out[:5], want) and (out[5:] == 7).all()
    got = ops.latent_attention_shared(ql, qr, s.batch.cache, **kw, scale=SCALE, out=ql)
    assert got.data_ptr() == ql.data_ptr() and torch.equal(ql, want)


def test_two_calls_give_the_same_bits_in_any_workspace(ops):
    print("[case] shared twice", flush=True)
    s = Shared([(3000, [(500, 1), (70, 2)]), (200, [(9, 1)])], 16, 64, True, 18)
    first = s.call(ops)
    need = ops.latent_attention_shared_workspace_bytes(2, 3, 4, 16)
    ws = torch.full((need + 256,), 0xa5, dtype=torch.uint8, device="cuda")
    again = s.call(ops, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and (ws[need:] == 0xa5).all()
    lib_native = lib.native()
    try:
        lib.native = lambda: lib._Absent()
        python = s.call(ops)
    finally:
        lib.native = lambda: lib_native
    assert all(torch.equal(a, b) for a, b in zip(first, python))


def test_another_stream_and_captured_replays(ops):
    """A captured call replays with other lengths, prefixes and queries."""
    print("[case] shared captured", flush=True)
    batch = [Shared([(p, [(a, 1), (b, 2)]), (q, [(c, 1)])], 16, 16, True, 19) for p, q, a, b, c in
             ((300, 64, 30, 65, 9), (17, 0, 1, 200, 64), (500, 130, 64, 2, 33))]
    most = max(s.batch.table.shape[1] for s in batch)
    pages = max(s.batch.pages for s in batch)
    eager = [s.call(ops) for s in batch]

    def state(s):
        kw = s.index()
        for name in ("prefix_table", "page_table"):
            wide = torch.full((kw[name].shape[0], most), -1, dtype=torch.int32, device="cuda")
            wide[:, :kw[name].shape[1]] = kw[name]
            kw[name] = wide
        data = torch.zeros((pages, 16, 640), dtype=torch.uint8, device="cuda")
        scales = torch.zeros((pages, 16, 4), dtype=torch.uint8, device="cuda")
        data[:s.batch.pages], scales[:s.batch.pages] = s.batch.cache.data, s.batch.cache.scales
        return dict(kw, ql=bf16_tensor(s.ql), qr=bf16_tensor(s.qr), data=data, scales=scales)

    states = [state(s) for s in batch]
    now = {k: v.clone() for k, v in states[0].items()}

    def call():
        kw = {k: v for k, v in now.items() if k not in ("ql", "qr", "data", "scales")}
        return ops.latent_attention_shared(now["ql"], now["qr"], ops.LatentCache(now["data"], now["scales"]), **kw,
                                           scale=SCALE, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out[0], eager[0][0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for i in (1, 2, 0, 2):
        for k, v in states[i].items():
            now[k].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        batch[i].check(*out)
        assert torch.equal(out[0], eager[i][0]) and torch.equal(out[1], eager[i][1]), i


def test_rows_past_32_bits_of_the_cache(ops):
    """The last pages of a cache of 9 GB: the bits of the small one."""
    print("[case] shared far pages", flush=True)
    for e4m3, H in ((True, 16), (False, 16), (True, 64), (False, 64)):
        s = Shared([(300, [(30, 1), (65, 4)])], H, 16, e4m3, 22)
        want, want_lse = s.call(ops)
        small = s.batch.cache
        pages = 9 * 2 ** 30 // (small.data.stride(0) * small.data.element_size())
        far, gap = ops.LatentCache.empty(pages, 16, small.data.dtype if not e4m3 else torch.float8_e4m3fn), pages - s.batch.pages
        far.data[gap:] = small.data
        if e4m3:
            far.scales[gap:] = small.scales
        kw = s.index()
        for name in ("prefix_table", "page_table"):
            kw[name] = torch.where(kw[name] >= 0, kw[name] + gap, kw[name])
        out, lse = ops.latent_attention_shared(bf16_tensor(s.ql), bf16_tensor(s.qr), far, **kw, scale=SCALE, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), (e4m3, H)
        del far


def test_two_calls_at_once(ops):
    """Two streams, each with calls of its own in flight."""
    print("[case] shared on two streams", flush=True)
    both = [Shared([(3000, [(500, 1), (70, 2)])], 16, 64, True, 23), Shared([(900, [(20, 1)] * 9)], 64, 16, False, 24)]
    want = [s.call(ops) for s in both]
    args = [(bf16_tensor(s.ql), bf16_tensor(s.qr), s.batch.cache, s.index()) for s in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (ql, qr, cache, kw) in enumerate(args):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.latent_attention_shared(ql, qr, cache, **kw, scale=SCALE, return_lse=True))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i]), i


def test_a_captured_prefix_pass(ops):
    """Prefixes in a pass of their own: replays with other lengths, missing pages and a NaN that stays with its prefix."""
    print("[case] shared captured, prefixes apart", flush=True)
    for e4m3 in (True, False):
        batch = [Shared([(p, [(a, 1)] * 3 + [(b, 1)]), (q, [(c, 1)] * 4)], 16, 16, e4m3, 25)
                 for p, q, a, b, c in ((300, 640, 30, 65, 9), (17, 0, 1, 200, 64), (5000, 1300, 64, 0, 33))]
        columns = max(s.wide()["prefix_table"].shape[1] for s in batch)
        own = max(s.batch.table.shape[1] for s in batch)
        pages = max(s.batch.pages for s in batch)

        def state(s):
            kw = s.index()
            for name, most in (("prefix_table", columns), ("page_table", own)):
                wide = torch.full((kw[name].shape[0], most), -1, dtype=torch.int32, device="cuda")
                wide[:, :kw[name].shape[1]] = kw[name][:, :most]
                kw[name] = wide
            cache = ops.LatentCache.empty(pages, 16, torch.float8_e4m3fn if e4m3 else torch.bfloat16)
            cache.data.zero_()
            cache.data[:s.batch.pages] = s.batch.cache.data
            if e4m3:
                cache.scales.fill_(127)
                cache.scales[:s.batch.pages] = s.batch.cache.scales
            return dict(kw, ql=bf16_tensor(s.ql), qr=bf16_tensor(s.qr), data=cache.data,
                        **({"scales": cache.scales} if e4m3 else {}))
        states = [state(s) for s in batch]
        now = {k: v.clone() for k, v in states[0].items()}

        def call(now):
            kw = {k: v for k, v in now.items() if k not in ("ql", "qr", "data", "scales")}
            return ops.latent_attention_shared(now["ql"], now["qr"], ops.LatentCache(now["data"], now.get("scales")), **kw,
                                               scale=SCALE, return_lse=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(now)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(now)
        for i in (1, 2, 0, 2):
            for k, v in states[i].items():
                now[k].copy_(v)
            g.replay()
            want = call(states[i])
            torch.cuda.synchronize()
            batch[i].check(*out)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
        bad = dict(states[0], data=states[0]["data"].clone())
        want = call(states[0])
        page = int(bad["prefix_table"][1, 3])
        if e4m3:
            bad["data"][page, 5, 70] = 0x7f
        else:
            bad["data"][page, 5, 70] = float("nan")
        got = call(bad)
        assert torch.isnan(got[0][4:]).all() and torch.equal(got[0][:4], want[0][:4])
        gone = dict(states[0], prefix_table=states[0]["prefix_table"].clone())
        gone["prefix_table"][0, 2] = -1
        got = call(gone)
        s = batch[0]
        keep = np.ones(300, dtype=bool)
        keep[32:48] = False
        s.batch.lat[0], s.batch.rot[0] = s.batch.lat[0][keep], s.batch.rot[0][keep]
        s.groups = [(284, s.groups[0][1]), s.groups[1]]
        s.check(*got)


def test_workspace_of_both_ways(ops):
    """One workspace size whatever the tables; nothing is written past it."""
    print("[case] shared workspaces", flush=True)
    s = Shared([(900, [(20, 1)] * 7)], 16, 16, True, 26)
    need = ops.latent_attention_shared_workspace_bytes(1, 7, 7, 16)
    for kw in (s.index(), s.wide()):
        ws = torch.full((need + 256,), 0xa5, dtype=torch.uint8, device="cuda")
        out = ops.latent_attention_shared(bf16_tensor(s.ql), bf16_tensor(s.qr), s.batch.cache, **kw, scale=SCALE,
                                          workspace=ws)
        again = s.call(ops, **kw)
        assert torch.equal(out, again[0]) and (ws[need:] == 0xa5).all()


@pytest.mark.parametrize("H,members", [(16, 4), (16, 8), (1, 9), (5, 40), (32, 2), (24, 5), (17, 30)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_prefixes_in_a_pass_of_their_own(ops, H, members, e4m3):
    """Full and ragged tiles of a prefix, cut in pieces and whole, beside short, long and missing own keys."""
    print(f"[case] shared prefix pass H={H} members={members} e4m3={e4m3}", flush=True)
    own = [(0, 1), (3000, 1), (65, 1), (1, 1), (64, 1), (200, 1)]
    s = Shared([(1700, [own[i % 6] for i in range(members)]), (0, [(40, 1)] * members), (63, [own[i % 4] for i in range(members)])],
               H, 16, e4m3, 27)
    assert s.wide() is not None
    s.run(ops)


def test_other_tokens_beside_a_prefix_pass(ops):
    """Sequences before and behind the prefixes, of several tokens, some not causal."""
    print("[case] shared prefix pass with others", flush=True)
    s = Shared([(None, [(90, 2), (7, 1)]), (500, [(30, 1), (2, 2), (64, 1), (9, 1)] * 3), (None, [(65, 1), (130, 1)])], 8, 16, True, 28)
    assert s.wide() is not None
    s.run(ops)
    s.run(ops, causal=False)
