"""GPU: latent attention in its absorbed form against the formula in 64 bits (oracle.attention),
with bounds that count every rounding (oracle.attention.bounds)."""
import numpy as np
import pytest
import torch

from oracle import formats as F
from tests.attention_helpers import SCALE, Batch, bf16_tensor, bf16_values, check_absorbed, i32, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


def _queries(T, H, seed, std=1.0):
    rng = np.random.default_rng(seed)
    return bf16_values(rng, T, H, 512, std=std), bf16_values(rng, T, H, 64, std=std)


def _run(ops, b, new, H, causal=True, scale=SCALE, seed=3, std=1.0, check=True):
    ql, qr = _queries(max(1, sum(new)), H, seed, std)
    table, lens = b.device()
    out, lse = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32(starts(new)), scale,
                                    causal=causal, return_lse=True)
    torch.cuda.synchronize()
    if check:
        worst = check_absorbed(b, new, ql, qr, out, lse, causal, scale)
        print(f"    worst {worst:.3f} of the bound", flush=True)
    return out, lse


@pytest.mark.parametrize("H", [1, 3, 16, 17, 32, 48, 64, 100, 128])
@pytest.mark.parametrize("e4m3", [False, True])
def test_one_token_per_sequence(ops, H, e4m3):
    """Lengths around the steps of 64 and the pages; one sequence long enough to be cut into pieces."""
    print(f"[case] absorbed decode H={H} e4m3={e4m3}", flush=True)
    lens = [1, 15, 16, 17, 63, 64, 65, 127, 130, 700]
    _run(ops, Batch(lens, 48, e4m3, H), [1] * len(lens), H)


@pytest.mark.parametrize("new", [[1], [2], [3, 0, 1, 40, 5], [64, 64], [70, 1]])
@pytest.mark.parametrize("H", [2, 16, 40])
@pytest.mark.parametrize("e4m3", [False, True])
def test_several_tokens_per_sequence(ops, new, H, e4m3):
    """Chunks: every token sees up to its own key; more new tokens than keys leave the first without any."""
    print(f"[case] absorbed chunk new={new} H={H} e4m3={e4m3}", flush=True)
    lens = [max(n + d, 0) for n, d in zip(new, (37, -1 if len(new) > 1 else 0, 100, 33, -3))]
    _run(ops, Batch(lens, 16, e4m3, 11), new, H)


@pytest.mark.parametrize("e4m3", [False, True])
def test_all_keys_visible(ops, e4m3):
    print(f"[case] absorbed non-causal e4m3={e4m3}", flush=True)
    _run(ops, Batch([70, 5, 0, 129], 32, e4m3, 4), [3, 7, 2, 1], 8, causal=False)


@pytest.mark.parametrize("H,lens", [(16, [9000]), (128, [2500, 1]), (64, [0, 5000]), (24, [1300, 40, 4100])])
@pytest.mark.parametrize("e4m3", [False, True])
def test_long_sequences_are_cut_and_joined(ops, H, lens, e4m3):
    print(f"[case] absorbed long H={H} lens={lens} e4m3={e4m3}", flush=True)
    _run(ops, Batch(lens, 64, e4m3, 6), [1] * len(lens), H)


def test_large_scores(ops):
    """Scores of some hundreds: the running maximum moves often, most terms vanish."""
    print("[case] absorbed large scores", flush=True)
    _run(ops, Batch([400, 1000], 64, False, 8), [2, 1], 16, std=8.0)
    _run(ops, Batch([400, 1000], 64, True, 8), [2, 1], 16, std=8.0)


def test_many_sequences(ops):
    """More sequences than a work-group has threads, most without new tokens."""
    print("[case] absorbed 600 sequences", flush=True)
    lens = [(7 * i) % 50 for i in range(600)]
    new = [1 if i % 5 == 0 else 0 for i in range(600)]
    _run(ops, Batch(lens, 16, True, 9), new, 4)


def test_strides_and_streams(ops):
    """Queries as transposed products and slices of wider tensors, on another stream with a workspace of its own."""
    print("[case] absorbed strides", flush=True)
    b, H, new = Batch([200, 77], 32, True, 2), 16, [1, 3]
    ql, qr = _queries(4, H, 3)
    table, lens = b.device()
    want = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32(starts(new)), SCALE)
    heads_first = bf16_tensor(ql).transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((4, H, 192), dtype=torch.bfloat16, device="cuda")
    wide[..., 128:] = bf16_tensor(qr)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.latent_attention(heads_first, wide[..., 128:], b.cache, table, lens, i32(starts(new)), SCALE)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_the_same_call_gives_the_same_bits(ops):
    print("[case] absorbed repeat", flush=True)
    b = Batch([3000, 500, 40], 64, True, 12)
    a = _run(ops, b, [1, 1, 1], 16, check=False)
    for _ in range(3):
        c = _run(ops, b, [1, 1, 1], 16, check=False)
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_rows_behind_the_last_sequence_stay(ops):
    print("[case] absorbed padded batch", flush=True)
    b, H = Batch([100, 30], 16, False, 1), 5
    ql, qr = _queries(9, H, 3)
    table, lens = b.device()
    out = torch.full((9, H, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    got, lse = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32([0, 2, 5]), SCALE,
                                    return_lse=True, out=out)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr() and (out[5:] == 7).all()
    check_absorbed(b, [2, 3], ql, qr, out, lse)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("H,new", [(16, [1, 1, 1]), (8, [20, 3, 90]), (128, [1, 2, 1])])
def test_nan_in_unused_slots_and_unseen_rows(ops, e4m3, H, new):
    """Every slot without a key holds NaN (and NaN scales); the bits are those of a clean cache.  A
    NaN among the new tokens' rows reaches the tokens that see it and no other."""
    print(f"[case] absorbed NaN e4m3={e4m3} H={H} new={new}", flush=True)
    lens = [100, 21, 130]
    clean, dirty = Batch(lens, 64, e4m3, 7), Batch(lens, 64, e4m3, 7, poison=True)
    a, la = _run(ops, clean, new, H, check=False)
    b, lb = _run(ops, dirty, new, H)
    assert torch.equal(a, b) and torch.equal(la, lb)
    row = int(dirty.slots[2][lens[2] - 2 if new[2] > 1 else lens[2] - 1])
    flat = dirty.cache.data.view(-1, dirty.cache.data.shape[-1])
    for value in (float("nan"), float("inf")):
        if e4m3:
            flat[row, 5] = 0x7F
        else:
            flat[row, 5] = value
        c, _ = _run(ops, dirty, new, H, check=False)
        first = sum(new) - (2 if new[2] > 1 else 1)
        assert torch.equal(c[:first], a[:first])
        if value != value or e4m3:
            assert c[first:].isnan().all()
        else:  # a score of +inf; at -inf the key has no weight
            ql, _ = _queries(sum(new), H, 3)
            assert c[first:][torch.from_numpy(ql[first:, :, 5] > 0).cuda()].isnan().all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_entries_that_are_no_page_are_left_out(ops, e4m3):
    """The keys of such an entry are masked; a sequence of nothing else gives zeros."""
    print(f"[case] absorbed bad pages e4m3={e4m3}", flush=True)
    H, new = 16, [1, 2, 1]
    b = Batch([100, 64, 40], 16, e4m3, 3, poison=True)
    gone = [list(range(16, 32)), list(range(48, 64)), list(range(40))]
    b.table[0, 1], b.table[1, 3], b.table[2, :3] = -1, b.pages, [2 ** 31 - 1, -2 ** 31, 10 ** 6]
    ql, qr = _queries(4, H, 3)
    table, lens = b.device()
    out, lse = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32(starts(new)), SCALE,
                                    return_lse=True)
    torch.cuda.synchronize()
    assert (out[3] == 0).all() and (lse[3] == -np.inf).all()
    from oracle import attention as A
    t = 0
    for i, n in enumerate(new[:2]):
        k = np.concatenate([b.lat[i], b.rot[i]], 1)
        see = np.arange(b.lens[i])[None] <= (b.lens[i] - n + np.arange(n))[:, None]
        see[:, gone[i]] = False
        for h in range(H):
            o, ref, spread, reach = A.attend(np.concatenate([ql[t:t + n, h], qr[t:t + n, h]], 1), k, b.lat[i], SCALE, see)
            eo, _ = A.bounds(o, ref, spread, reach, 576, b.lens[i])
            assert (np.abs(out[t:t + n, h].float().cpu().numpy() - o) <= eo).all()
        t += n


def test_lengths_past_the_table_are_cut(ops):
    print("[case] absorbed lengths past the table", flush=True)
    b = Batch([64, 32], 16, False, 3)
    ql, qr = _queries(2, 4, 3)
    table, lens = b.device()
    table[1, 2:] = table[0, :2]   # the second sequence fills its table
    args = (bf16_tensor(ql), bf16_tensor(qr), b.cache, table)
    want = ops.latent_attention(*args, i32([64, 64]), i32([0, 1, 2]), SCALE)
    got = ops.latent_attention(*args, i32([2 ** 31 - 1, 65]), i32([0, 1, 2]), SCALE)
    none = ops.latent_attention(*args, i32([-5, 0]), i32([0, 1, 2]), SCALE)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and (none == 0).all()


def test_offsets_past_32_bits(ops):
    print("[case] absorbed cache of 5 GB", flush=True)
    for e4m3 in (False, True):
        width = 640 if e4m3 else 1152
        b = Batch([200, 90], 64, e4m3, 5)
        pages = 5 * 2 ** 30 // (64 * width)
        big = ops.LatentCache.empty(pages, 64, torch.float8_e4m3fn if e4m3 else torch.bfloat16)
        big.data[-b.pages:] = b.cache.data
        if e4m3:
            big.scales[-b.pages:] = b.cache.scales
        table, lens = b.device()
        ql, qr = (bf16_tensor(x) for x in _queries(2, 16, 3))
        want = ops.latent_attention(ql, qr, b.cache, table, lens, i32([0, 1, 2]), SCALE)
        got = ops.latent_attention(ql, qr, big, table + (pages - b.pages), lens, i32([0, 1, 2]), SCALE)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del big
        torch.cuda.empty_cache()


def test_captured_and_replayed_with_other_lengths(ops):
    """Two graphs with workspaces of their own, replayed in turn with lengths and tables changed in place."""
    print("[case] absorbed graphs", flush=True)
    H, B = 16, 3
    b = Batch([900, 300, 500], 64, True, 21)
    table, lens = b.device()
    cu = i32([0, 1, 2, 3])
    ql, qr = (bf16_tensor(x) for x in _queries(B, H, 3))
    calls = [lambda w, k=k: ops.latent_attention(ql, qr, b.cache, table, lens, cu, SCALE * (k + 1), return_lse=True,
                                                 workspace=w) for k in range(2)]
    need = ops.latent_attention_workspace_bytes(B, B, H)
    spaces = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c, w in zip(calls, spaces):
            c(w)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c, w in zip(calls, spaces):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c(w))
        graphs.append(g)
    for rep, now in enumerate(([900, 300, 500], [1, 299, 64], [640, 0, 450], [900, 1, 1])):
        lens.copy_(i32(now))
        for w in spaces:
            w.fill_(255)            # NaN wherever it is read as a number
        for g in graphs:
            g.replay()
        want = [c(None) for c in calls]
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1]), rep


def test_refusals(ops):
    b = Batch([40, 20], 16, False, 1)
    table, lens = b.device()
    ql, qr = (bf16_tensor(x) for x in _queries(2, 4, 1))
    cu = i32([0, 1, 2])
    with pytest.raises(ValueError, match="q_latent must be"):
        ops.latent_attention(ql[..., :256], qr, b.cache, table, lens, cu, SCALE)
    with pytest.raises(ValueError, match="q_rotary must be"):
        ops.latent_attention(ql, qr[:, :2], b.cache, table, lens, cu, SCALE)
    with pytest.raises(TypeError):
        ops.latent_attention(ql.half(), qr, b.cache, table, lens, cu, SCALE)
    with pytest.raises(TypeError):
        ops.latent_attention(ql, qr, b.cache, table, lens.long(), cu, SCALE)
    with pytest.raises(ValueError, match="page_table"):
        ops.latent_attention(ql, qr, b.cache, table[:1], lens, cu, SCALE)
    with pytest.raises(ValueError, match="out must have shape"):
        ops.latent_attention(ql, qr, b.cache, table, lens, cu, SCALE, out=ql[:1])
    with pytest.raises(ValueError, match="packed"):
        ops.latent_attention(ql.transpose(1, 2).contiguous().transpose(1, 2), qr, b.cache, table, lens, cu, SCALE)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="code -2"):
            ops.latent_attention(ql, qr, b.cache, table, lens, cu, scale)


@pytest.mark.parametrize("by", [80, -80])
@pytest.mark.parametrize("H", [16, 32, 64, 128])
def test_powers_of_two_go_through(ops, H, by):
    """Latents times 2^by (in the scale bytes) under queries times 2^-by: outputs times 2^by, bit for bit."""
    print(f"[case] absorbed e4m3, latents times 2^{by}, H={H}", flush=True)
    b, cu_q = Batch([700, 65, 130], 64, True, 17), i32([0, 1, 2, 3])
    (ql, qr), (table, lens) = _queries(3, H, 5), b.device()
    want = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, cu_q, SCALE)
    moved = ops.LatentCache(b.cache.data, (b.cache.scales.int() + by).clamp(0, 254).to(torch.uint8))
    got = ops.latent_attention(bf16_tensor(ql * np.float32(2.0 ** -by)), bf16_tensor(qr), moved, table, lens, cu_q, SCALE)
    torch.cuda.synchronize()
    assert torch.equal(got.float(), want.float() * 2.0 ** by)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("H", [16, 64])
def test_pages_shared_by_sequences_and_named_twice(ops, H, e4m3):
    print(f"[case] absorbed, shared pages e4m3={e4m3} H={H}", flush=True)
    b = Batch([158, 200, 64], 64, e4m3, 23)
    b.table[1, :2] = b.table[0, :2]               # a common prefix of 128 keys
    b.table[1, 2] = b.table[0, 0]                 # and its first page once more
    for x in (b.lat, b.rot):
        x[1] = np.concatenate([x[0][:128], x[0][:64], x[1][192:]])
    _run(ops, b, [3, 2, 1], H)


def test_two_calls_at_once(ops):
    """Calls that overlap on two streams, each with a workspace from the allocator, and one passed to both in turn."""
    print("[case] absorbed, two streams", flush=True)
    cases = [(Batch([3000, 900], 64, True, 31), 16), (Batch([500, 2000], 64, False, 32), 64)]
    args, want = [], []
    for b, H in cases:
        (ql, qr), (table, lens) = _queries(2, H, 9), b.device()
        args.append((bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32([0, 1, 2]), SCALE))
        want.append(ops.latent_attention(*args[-1]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(20):
        for s, a, g in zip(streams, args, got):
            with torch.cuda.stream(s):
                g.append(ops.latent_attention(*a))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)
    ws = torch.empty(max(ops.latent_attention_workspace_bytes(2, 2, H) for _, H in cases), dtype=torch.uint8, device="cuda")
    for _ in range(3):
        for a, w in zip(args, want):
            assert torch.equal(ops.latent_attention(*a, workspace=ws), w)
