"""GPU: latent attention over batches of one long sequence among short ones: its rows have many times the pieces of the
others and are joined by work-groups of their own.  Against the formula in 64 bits, as the even batches are."""
import numpy as np
import pytest
import torch

from oracle import attention as A
from tests.attention_helpers import SCALE, Batch, assert_near, bf16_tensor, bf16_values, check_absorbed, i32, starts
from tests.test_gpu_shared_attention import Shared

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


def queries(T, H, seed):
    rng = np.random.default_rng(seed)
    return bf16_values(rng, T, H, 512), bf16_values(rng, T, H, 64)


def one_long(B, at, long, short=40):
    lens = [short + 3 * i for i in range(B)]
    lens[at] = long
    return lens


@pytest.mark.parametrize("B,H,at,long", [(16, 16, 3, 9000), (32, 16, 31, 12000), (50, 16, 0, 12000), (9, 3, 4, 8000),
                                         (20, 5, 10, 6000), (24, 32, 7, 7000), (6, 64, 2, 6000), (5, 128, 4, 4100),
                                         (140, 16, 77, 9000)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_one_long_sequence(ops, B, H, at, long, e4m3):
    print(f"[case] skewed B={B} H={H} at={at} long={long} e4m3={e4m3}", flush=True)
    b = Batch(one_long(B, at, long), 64, e4m3, B + H)
    ql, qr = queries(B, H, 3)
    table, lens = b.device()
    out, lse = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32(starts([1] * B)), SCALE,
                                    return_lse=True)
    torch.cuda.synchronize()
    print(f"    worst {check_absorbed(b, [1] * B, ql, qr, out, lse):.3f} of the bound", flush=True)


@pytest.mark.parametrize("e4m3", [False, True])
def test_several_long_ones_and_ragged_tiles(ops, e4m3):
    """Long sequences side by side and apart, several tokens in tiles that are not full, some without any."""
    print(f"[case] skewed several e4m3={e4m3}", flush=True)
    lens = [20, 5000, 4800, 7, 0, 300, 6100, 64, 1, 90, 50, 33]
    new = [1, 2, 1, 3, 1, 0, 3, 1, 1, 2, 1, 1]
    for H in (5, 16):
        b = Batch(lens, 32, e4m3, 8)
        ql, qr = queries(sum(new), H, 4)
        table, cached = b.device()
        out, lse = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, cached, i32(starts(new)), SCALE,
                                        return_lse=True)
        torch.cuda.synchronize()
        check_absorbed(b, new, ql, qr, out, lse)


def test_replays_with_the_long_one_elsewhere(ops):
    """A captured call whose long sequence moves, vanishes and comes back, in place on the queries; rows behind the last
    sequence are left alone."""
    print("[case] skewed captured", flush=True)
    B, H = 24, 16
    batches = [Batch(one_long(B, at, long), 64, True, 30 + at) for at, long in ((2, 9000), (23, 9000), (5, 30), (11, 5000))]
    most, pages = max(b.table.shape[1] for b in batches), max(b.pages for b in batches)
    q = [queries(B + 2, H, 40 + i) for i in range(len(batches))]

    def state(b, ql, qr):
        table = torch.full((B, most), -1, dtype=torch.int32, device="cuda")
        table[:, :b.table.shape[1]] = torch.from_numpy(b.table).cuda()
        cache = ops.LatentCache.empty(pages, 64, torch.float8_e4m3fn)
        cache.data[:b.pages], cache.scales[:b.pages] = b.cache.data, b.cache.scales
        return [bf16_tensor(ql), bf16_tensor(qr), cache.data, cache.scales, table, i32(b.lens)]

    states, cu = [state(b, *x) for b, x in zip(batches, q)], i32(starts([1] * B))
    now = [t.clone() for t in states[0]]
    ws = torch.full((ops.latent_attention_workspace_bytes(B, B + 2, H) + 256,), 0x7f, dtype=torch.uint8, device="cuda")

    def call(s, **kw):
        return ops.latent_attention(s[0], s[1], ops.LatentCache(s[2], s[3]), s[4], s[5], cu, SCALE, return_lse=True, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(now, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = call(now, workspace=ws, out=now[0])
    assert out.data_ptr() == now[0].data_ptr()
    for i in (1, 2, 0, 3, 2, 1):
        for to, v in zip(now, states[i]):
            to.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        want, want_lse = call(states[i])
        check_absorbed(batches[i], [1] * B, q[i][0], q[i][1], out, lse)
        assert torch.equal(out[:B], want[:B]) and torch.equal(lse[:B], want_lse[:B]), i
        assert torch.equal(out[B:], states[i][0][B:]) and (ws[-256:] == 0x7f).all()


GROUPS = {
    "long own keys": [(300, [(40, 1), (9000, 1), (7, 1), (30, 1), (64, 1), (1, 1), (0, 1), (90, 1)])],
    "a long prefix": [(64, [(5, 1)] * 8), (9000, [(40, 1)] * 8), (200, [(9, 1)] * 8)],
    "both": [(64, [(5, 1)] * 8), (9000, [(40, 1), (6000, 1), (3, 1), (8, 1), (100, 1), (65, 1), (0, 1), (9, 1)]),
             (200, [(9, 1)] * 8)],
}


@pytest.mark.parametrize("name,H", [("long own keys", 16), ("a long prefix", 5), ("long own keys", 32), ("both", 16)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_shared_prefixes(ops, name, H, e4m3):
    """In one pass and with prefixes in a pass of their own, whose pieces are joined with those of the own keys."""
    print(f"[case] skewed shared {name} H={H} e4m3={e4m3}", flush=True)
    s = Shared(GROUPS[name], H, 64, e4m3, H)
    assert s.wide() is not None
    s.run(ops)


@pytest.mark.parametrize("H,members", [(16, 70), (32, 45)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_many_sequences_behind_two_prefixes(ops, H, members, e4m3):
    """Few pieces on average in both passes, many of one prefix and of one sequence: rows with many of either, of both
    and of none.  Some sequences against the formula, all against latent_attention over joined tables."""
    print(f"[case] skewed shared, many sequences H={H} members={members} e4m3={e4m3}", flush=True)
    page, long = 64, members // 3
    groups = [(8960, [(20 + i % 50, 1) for i in range(members)]), (64, [(1 + i % 70, 1) for i in range(members)])]
    groups[0][1][long] = (20000, 1)
    groups[1][1][5] = (30000, 1)
    s = Shared(groups, H, page, e4m3, H)
    assert s.wide() is not None
    out, lse = s.call(ops, **s.wide())
    kw = s.index()
    table = torch.full((2 * members, 140 + kw["page_table"].shape[1]), -1, dtype=torch.int32, device="cuda")
    for g, pages in ((0, 140), (1, 1)):
        lines = slice(g * members, (g + 1) * members)
        table[lines, :pages] = kw["prefix_table"][g, :pages]
        table[lines, pages:pages + kw["page_table"].shape[1]] = kw["page_table"][lines]
    lens = kw["lens"] + torch.tensor([8960] * members + [64] * members, dtype=torch.int32, device="cuda")
    ref = ops.latent_attention(bf16_tensor(s.ql), bf16_tensor(s.qr), s.batch.cache, table, lens, kw["cu_q"], SCALE)
    torch.cuda.synchronize()
    assert (out.float() - ref.float()).abs().max() < 2 ** -6 * ref.float().abs().max()
    out, lse = out.float().cpu().numpy(), lse.cpu().numpy()
    for b in (0, long, members - 1, members, members + 5, 2 * members - 1):
        g = b // members
        lat = np.concatenate([s.batch.lat[g], s.batch.lat[2 + b]])
        k = np.concatenate([lat, np.concatenate([s.batch.rot[g], s.batch.rot[2 + b]])], 1)
        see = np.ones((1, len(k)), dtype=bool)
        for h in range(0, H, 5):
            q = np.concatenate([s.ql[b:b + 1, h], s.qr[b:b + 1, h]], 1)
            o, ref_l, spread, reach = A.attend(q, k, lat, SCALE, see)
            eo, el = A.bounds(o, ref_l, spread, reach, 576, len(k))
            assert_near(out[b:b + 1, h], o, eo, f"seq {b} head {h}")
            assert_near(lse[b:b + 1, h], ref_l, el, f"lse seq {b} head {h}")
