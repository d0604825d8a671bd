"""GPU: latent attention over shared prefixes whose prefixes get a pass of their own, at the edges: every call here asks
that it did take two passes (only they write behind the first 64 MiB of the workspace)."""
import numpy as np
import pytest
import torch

from ferret_amd import lib
from tests.attention_helpers import SCALE, bf16_tensor, i32
from tests.test_gpu_shared_attention import Shared

pytestmark = pytest.mark.gpu

FILL = 0xa5
APART = 64 << 20  # past what one pass writes in tiles of 16 or 32 rows, before the second pass's records


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


def two_passes(ops, s, ql=None, qr=None, cache=None, kw=None, **more):
    """(out, lse) of a call that is checked to have taken two passes and to have stayed inside its workspace."""
    ql, qr = bf16_tensor(s.ql) if ql is None else ql, bf16_tensor(s.qr) if qr is None else qr
    kw = s.wide() if kw is None else kw
    assert kw is not None, "the rows allow no pass for the prefixes"
    G, B = kw["prefix_lens"].numel(), kw["lens"].numel()
    need = ops.latent_attention_shared_workspace_bytes(G, B, ql.shape[0], ql.shape[1])
    ws = torch.full((need + 256,), FILL, dtype=torch.uint8, device="cuda")
    got = ops.latent_attention_shared(ql, qr, s.batch.cache if cache is None else cache, **kw, scale=SCALE,
                                      return_lse=True, workspace=ws, **more)
    assert (ws[APART:need] != FILL).any(), "one pass"
    assert (ws[need:] == FILL).all()
    return got


def test_one_pass_stays_before_them(ops):
    """What the check above rests on."""
    print("[case] shared one pass's workspace", flush=True)
    s = Shared([(300, [(30, 1)] * 8)], 16, 16, True, 1)
    need = ops.latent_attention_shared_workspace_bytes(1, 8, 8, 16)
    ws = torch.full((need,), FILL, dtype=torch.uint8, device="cuda")
    s.check(*s.call(ops, workspace=ws))
    assert (ws[:APART] != FILL).any() and (ws[APART:] == FILL).all()


@pytest.mark.parametrize("H", [5, 16, 32])
@pytest.mark.parametrize("e4m3", [False, True])
def test_unseen_rows_do_not_reach(ops, H, e4m3):
    """NaN in every slot that no key has, the ends of the prefixes' pages among them."""
    print(f"[case] two passes, poisoned slots H={H} e4m3={e4m3}", flush=True)
    s = Shared([(75, [(20, 1), (33, 1), (1, 1), (0, 1)] * 2), (130, [(1, 1), (64, 1)] * 4), (0, [(0, 1), (17, 1)] * 4)], H, 48,
               e4m3, 12, poison=True)
    out, lse = two_passes(ops, s)
    s.check(out, lse)
    assert (out[16] == 0).all() and torch.isneginf(lse[16]).all()


@pytest.mark.parametrize("H", [5, 16, 32])
def test_latents_past_448(ops, H):
    """Exponent bytes above 127 in some rows and blocks of 128 latents, in prefix and own keys."""
    print(f"[case] two passes, large latents H={H}", flush=True)
    s = Shared([(200, [(90, 1), (40, 1)] * 4)], H, 16, True, 20)
    scales = s.batch.cache.scales.view(-1, 4)
    rng = np.random.default_rng(21)
    byte = scales.cpu().numpy()
    for line, slots in enumerate(s.batch.slots):
        more = rng.integers(1, 7, (len(slots), 4)) * (rng.random((len(slots), 4)) < 0.1)
        byte[slots] += more.astype(np.uint8)
        s.batch.lat[line] = s.batch.lat[line] * np.repeat(np.exp2(more), 128, axis=1)
    assert (byte > 127).any()
    scales.copy_(torch.from_numpy(byte))
    s.ql = s.ql * 2.0 ** -9
    s.check(*two_passes(ops, s))


@pytest.mark.parametrize("e4m3", [False, True])
def test_lengths_past_the_tables_and_below_zero(ops, e4m3):
    """Lengths are cut to the tables, negative ones are none; entries past a prefix's own pages are none."""
    print(f"[case] two passes, lengths out of range e4m3={e4m3}", flush=True)
    s = Shared([(64, [(32, 1)] * 4), (48, [(16, 1)] * 4)], 16, 16, e4m3, 15)
    kw = s.wide()
    kw["prefix_lens"] = i32([1 << 30, -7])
    kw["lens"] = i32([1 << 30, 32, 32, 32, -5, 16, 16, 16])
    out, lse = two_passes(ops, s, kw=kw)
    s.groups = [(64, [(32, 1)] * 4), (0, [(0, 1)] + [(16, 1)] * 3)]
    for line in (1, 6):
        s.batch.lat[line], s.batch.rot[line] = s.batch.lat[line][:0], s.batch.rot[line][:0]
    s.check(out, lse)
    assert (out[4] == 0).all() and torch.isneginf(lse[4]).all()


@pytest.mark.parametrize("H", [16, 32])
@pytest.mark.parametrize("e4m3", [False, True])
def test_strides_places_and_rows_behind(ops, H, e4m3):
    """Queries head by head and inside a wider projection, an output in place on packed queries, and rows behind the last
    sequence left alone."""
    print(f"[case] two passes, strides H={H} e4m3={e4m3}", flush=True)
    s = Shared([(300, [(30, 1), (65, 1), (0, 1), (64, 1)] * 2)], H, 16, e4m3, 17)
    want, want_lse = two_passes(ops, s)
    s.check(want, want_lse)
    ql, qr = bf16_tensor(s.ql), bf16_tensor(s.qr)
    T = ql.shape[0]
    heads = ql.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((T, H, 192), dtype=torch.bfloat16, device="cuda")
    wide[..., 128:] = qr
    out, lse = two_passes(ops, s, heads, wide[..., 128:])
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    place = ql.clone()
    out, lse = two_passes(ops, s, place, out=place)
    assert out.data_ptr() == place.data_ptr() and torch.equal(place, want) and torch.equal(lse, want_lse)
    # rows behind: in tiles by the rows that a sequence has with them
    if H == 16:
        out = torch.full((T + 3, H, 512), 7.0, dtype=torch.bfloat16, device="cuda")
        got, lse = two_passes(ops, s, torch.cat([ql, ql[:3]]), torch.cat([qr, qr[:3]]), out=out)
        s.check(got[:T], lse[:T])
        assert got.data_ptr() == out.data_ptr() and (out[T:] == 7).all()
    # and before the first: nobody's tokens
    kw = s.wide()
    kw["cu_q"], kw["cu_prefix"] = kw["cu_q"] + 1, kw["cu_prefix"] + 1
    if H == 16:
        kw = {**kw, "prefix_table": torch.cat([kw["prefix_table"], kw["prefix_table"].new_full((1, 4000), -1)], 1)}
        out = torch.full((T + 1, H, 512), 7.0, dtype=torch.bfloat16, device="cuda")
        got, lse = two_passes(ops, s, torch.cat([ql[:1], ql]), torch.cat([qr[:1], qr]), kw=kw, out=out)
        s.check(got[1:], lse[1:])
        assert (out[0] == 7).all()


@pytest.mark.parametrize("H", [16, 32])
@pytest.mark.parametrize("e4m3", [False, True])
def test_rows_past_32_bits_of_the_cache(ops, H, e4m3):
    """The last pages of a cache of 9 GB: the bits of the small one."""
    print(f"[case] two passes, far pages H={H} e4m3={e4m3}", flush=True)
    s = Shared([(300, [(30, 1), (65, 1)] * 4)], H, 16, e4m3, 22)
    want, want_lse = two_passes(ops, s)
    s.check(want, want_lse)
    small = s.batch.cache
    pages = 9 * 2 ** 30 // (small.data.stride(0) * small.data.element_size())
    far, gap = ops.LatentCache.empty(pages, 16, torch.float8_e4m3fn if e4m3 else torch.bfloat16), pages - s.batch.pages
    far.data[gap:] = small.data
    if e4m3:
        far.scales[gap:] = small.scales
    kw = s.wide()
    for name in ("prefix_table", "page_table"):
        kw[name] = torch.where(kw[name] >= 0, kw[name] + gap, kw[name])
    out, lse = two_passes(ops, s, cache=far, kw=kw)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_two_calls_at_once(ops):
    """Two streams, each with two-pass calls of its own in flight."""
    print("[case] two passes on two streams", flush=True)
    both = [Shared([(1500, [(500, 1), (70, 1)] * 4)], 16, 64, True, 23), Shared([(900, [(20, 1)] * 9), (64, [(7, 1)] * 9)], 5, 16,
                                                                                False, 24)]
    want = [two_passes(ops, s) for s in both]
    for s, w in zip(both, want):
        s.check(*w)
    args = [(bf16_tensor(s.ql), bf16_tensor(s.qr), s.batch.cache, s.wide()) for s in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (ql, qr, cache, kw) in enumerate(args):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.latent_attention_shared(ql, qr, cache, **kw, scale=SCALE, return_lse=True))
    torch.cuda.synchronize()
    for w, calls in zip(want, got):
        assert all(torch.equal(o, w[0]) and torch.equal(l, w[1]) for o, l in calls)


def test_the_same_bits_in_any_workspace_and_from_python(ops, monkeypatch):
    print("[case] two passes twice", flush=True)
    s = Shared([(1500, [(500, 1), (70, 1), (9, 1), (0, 1)]), (200, [(9, 1)] * 4)], 16, 64, True, 18)
    first = two_passes(ops, s)
    s.check(*first)
    kw, ql, qr = s.wide(), bf16_tensor(s.ql), bf16_tensor(s.qr)
    again = ops.latent_attention_shared(ql, qr, s.batch.cache, **kw, scale=SCALE, return_lse=True)
    small = ops.latent_attention_shared(ql, qr, s.batch.cache, **kw, scale=SCALE, return_lse=True,
                                        workspace=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
    index = [kw[k] for k in ("prefix_table", "prefix_lens", "cu_prefix", "page_table", "lens", "cu_q")]
    assert lib.native().latent_attention_shared(ql, qr, s.batch.cache.data, s.batch.cache.scales, *index, SCALE, True, True,
                                                None, None) is not None
    monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    python = two_passes(ops, s)
    for other in (again, small, python):
        assert torch.equal(other[0], first[0]) and torch.equal(other[1], first[1])
    import ferret_amd.torch_ops  # noqa: F401
    o, lse = torch.ops.ferret.latent_attention_shared(ql, qr, s.batch.cache.data, s.batch.cache.scales, *index, SCALE, True)
    assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


@pytest.mark.parametrize("e4m3", [False, True])
def test_nan_stays_with_its_tokens(ops, e4m3):
    """In one prefix, and in one sequence's own keys."""
    print(f"[case] two passes, NaN e4m3={e4m3}", flush=True)
    s = Shared([(100, [(9, 1)] * 4), (100, [(30, 1)] * 4)], 16, 16, e4m3, 13)
    want, _ = two_passes(ops, s)
    data = s.batch.cache.data.view(s.batch.pages * 16, -1)
    saved = data.clone()

    def plant(line, at):
        data.copy_(saved)
        data[s.batch.slots_of(line, at + 1)[at], 5] = 0x7f if e4m3 else float("nan")
        return two_passes(ops, s)[0]

    got = plant(0, 41)
    assert torch.isnan(got[:4]).all() and torch.equal(got[4:], want[4:])
    got = plant(2 + 6, 29)      # the last key of sequence 6
    others = [i for i in range(8) if i != 6]
    assert torch.isnan(got[6]).all() and torch.equal(got[others], want[others])


@pytest.mark.parametrize("e4m3", [False, True])
def test_no_tokens_behind_the_prefixes(ops, e4m3):
    """All of the work-groups go to the sequences where no token sees a prefix, all to the prefixes where the sequences'
    keys are none, and where there are no tokens nothing is written."""
    print(f"[case] two passes, none of one line e4m3={e4m3}", flush=True)
    s = Shared([(300, [(30, 1), (65, 1), (0, 1), (64, 1)]), (75, [(7, 1)] * 4)], 16, 16, e4m3, 31)
    kw = s.wide()
    for none in ([0, 0, 0], [4, 4, 4], [8, 8, 8]):
        out, lse = two_passes(ops, s, kw={**kw, "cu_prefix": i32(none)})
        want = ops.latent_attention(bf16_tensor(s.ql), bf16_tensor(s.qr), s.batch.cache, kw["page_table"], kw["lens"],
                                    kw["cu_q"], SCALE, return_lse=True)
        alone = Shared([(None, s.own)], 16, 16, e4m3, 31)
        alone.batch, alone.ql, alone.qr, alone.G = s.batch, s.ql, s.qr, 2
        alone.check(out, lse)
        alone.check(*want)
    out, lse = two_passes(ops, s, kw={**kw, "lens": i32([0] * 8)})
    s.groups = [(300, [(0, 1)] * 4), (75, [(0, 1)] * 4)]
    for line in range(2, 10):
        s.batch.lat[line], s.batch.rot[line] = s.batch.lat[line][:0], s.batch.rot[line][:0]
    s.check(out, lse)
    out = torch.full((8, 16, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    two = {**kw, "cu_q": i32([0] * 9), "cu_prefix": i32([0] * 3)}
    ops.latent_attention_shared(bf16_tensor(s.ql), bf16_tensor(s.qr), s.batch.cache, **two, scale=SCALE, out=out)
    assert (out == 7).all()
