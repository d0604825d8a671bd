"""GPU: latent attention in its expanded form against the formula in 64 bits, with bounds that
count every rounding (oracle.attention.bounds)."""
import numpy as np
import pytest
import torch

from oracle import attention as A
from tests.attention_helpers import SCALE, assert_near, bf16_tensor, bf16_values, i32, starts, visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


class Case:
    def __init__(self, lens, new, H, seed=0, std=1.0, spare=0):
        rng = np.random.default_rng(seed + H + sum(lens))
        T, S = sum(new) + spare, sum(lens) + spare
        self.lens, self.new, self.H = lens, new, H
        self.qn, self.qr = bf16_values(rng, T, H, 128, std=std), bf16_values(rng, T, H, 64, std=std)
        self.kn, self.kr = bf16_values(rng, S, H, 128), bf16_values(rng, S, 64)
        self.v = bf16_values(rng, S, H, 128)

    def tensors(self):
        kv = bf16_tensor(np.concatenate([self.kn, self.v], -1))       # as the key-value projection gives it
        q = bf16_tensor(np.concatenate([self.qn, self.qr], -1))
        return q[..., :128], q[..., 128:], kv[..., :128], bf16_tensor(self.kr), kv[..., 128:]

    def run(self, ops, causal=True, **kw):
        out = ops.latent_attention_expanded(*self.tensors(), i32(starts(self.new)), i32(starts(self.lens)), SCALE,
                                            causal=causal, return_lse=True, **kw)
        torch.cuda.synchronize()
        return out

    def check(self, out, lse, causal=True):
        out, lse = out.float().cpu().numpy(), lse.cpu().numpy()
        t = k0 = 0
        worst = 0.0
        for b, (length, n) in enumerate(zip(self.lens, self.new)):
            see = visible(n, length, causal)
            for h in range(self.H):
                q = np.concatenate([self.qn[t:t + n, h], self.qr[t:t + n, h]], 1)
                k = np.concatenate([self.kn[k0:k0 + length, h], self.kr[k0:k0 + length]], 1)
                o, ref, spread, reach = A.attend(q, k, self.v[k0:k0 + length, h], SCALE, see)
                eo, el = A.bounds(o, ref, spread, reach, 192, length)
                worst = max(worst, assert_near(out[t:t + n, h], o, eo, f"seq {b} head {h}"))
                assert_near(lse[t:t + n, h], ref, el, f"lse seq {b} head {h}")
            t, k0 = t + n, k0 + length
        print(f"    worst {worst:.3f} of the bound", flush=True)


@pytest.mark.parametrize("lens,new", [([1], [1]), ([5], [5]), ([64, 65], [64, 1]), ([130, 0, 40, 16], [128, 0, 33, 17]),
                                      ([300, 129], [129, 129]), ([20, 10], [23, 12]), ([700], [3])])
@pytest.mark.parametrize("H", [1, 3, 16])
def test_ragged(ops, lens, new, H):
    print(f"[case] expanded lens={lens} new={new} H={H}", flush=True)
    c = Case(lens, new, H)
    c.check(*c.run(ops))


def test_all_keys_visible(ops):
    print("[case] expanded non-causal", flush=True)
    c = Case([70, 5, 0, 129], [3, 140, 2, 1], 4)
    c.check(*c.run(ops, causal=False), causal=False)


def test_large_scores(ops):
    print("[case] expanded large scores", flush=True)
    c = Case([300, 200], [200, 60], 4, std=12.0)
    c.check(*c.run(ops))


def test_many_sequences(ops):
    print("[case] expanded 150 sequences", flush=True)
    new = [(3 * i) % 7 for i in range(150)]
    c = Case([n + i % 5 for i, n in enumerate(new)], new, 2)
    c.check(*c.run(ops))


def test_a_longer_prompt(ops):
    print("[case] expanded 1500 of 2000", flush=True)
    c = Case([2000], [1500], 2)
    c.check(*c.run(ops))


def test_padded_rows_strides_and_streams(ops):
    print("[case] expanded padded", flush=True)
    c = Case([100, 30], [60, 20], 4, spare=9)
    out = torch.full((89, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got, lse = c.run(ops, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[80:] == 7).all()
    c.check(out, lse)
    qn, qr, kn, kr, v = c.tensors()
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (qn, qr, kn, v)]
    wide = torch.cat([kr, kr], 1)[:, 64:]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = ops.latent_attention_expanded(heads_first[0], heads_first[1], heads_first[2], wide, heads_first[3],
                                              i32(starts(c.new)), i32(starts(c.lens)), SCALE)
    torch.cuda.synchronize()
    assert torch.equal(again[:80], out[:80])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_that_a_token_does_not_see(ops, value):
    """Inf or NaN among the values reaches its own column of the tokens that see it; among the
    keys, the tokens that see it; and nothing else."""
    print(f"[case] expanded {value}", flush=True)
    c = Case([150, 40], [140, 40], 2)
    clean, _ = c.run(ops)
    c.v[100, 1, 17] = value                       # key 100 of the first sequence: new token 90
    out, _ = c.run(ops)
    got, want = out.float(), clean.float()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[90:140, 1, 17] = True
    assert torch.equal(got[~hit], want[~hit])
    if value != value:
        assert got[hit].isnan().all()
    else:
        assert (got[hit] == value).all()
    c = Case([150, 40], [140, 40], 2)
    c.kn[150 + 25, 0, 3] = float("nan")           # key 25 of the second, seen from its own token on
    out, _ = c.run(ops)
    got, hit = out.float(), torch.zeros_like(want, dtype=torch.bool)
    hit[140 + 25:, 0] = True
    assert torch.equal(got[~hit], want[~hit]) and got[hit].isnan().all()


def test_the_same_call_gives_the_same_bits_and_replays(ops):
    print("[case] expanded graph", flush=True)
    c = Case([400, 300], [300, 300], 4)
    args = c.tensors()
    cu_q, cu_k = i32(starts(c.new)), i32(starts(c.lens))

    def call():
        return ops.latent_attention_expanded(*args, cu_q, cu_k, SCALE, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for new, lens in (([300, 300], [400, 300]), ([10, 500], [100, 600]), ([0, 600], [0, 700])):
        cu_q.copy_(i32(starts(new)))
        cu_k.copy_(i32(starts(lens)))
        g.replay()
        want = call()
        torch.cuda.synchronize()
        rows = sum(new)                 # what stands behind the last sequence is not set
        assert torch.equal(got[0][:rows], want[0][:rows]) and torch.equal(got[1][:rows], want[1][:rows])


def test_index_values_outside_the_tensors_are_cut(ops):
    print("[case] expanded index values", flush=True)
    c = Case([50, 40], [30, 40], 2)
    args = c.tensors()
    want = ops.latent_attention_expanded(*args, i32([0, 30, 70]), i32([0, 50, 90]), SCALE)
    got = ops.latent_attention_expanded(*args, i32([-7, 30, 2 ** 31 - 1]), i32([-2 ** 31, 50, 1000]), SCALE)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_refusals(ops):
    c = Case([40], [40], 4)
    qn, qr, kn, kr, v = c.tensors()
    cu = i32([0, 40])
    with pytest.raises(ValueError, match="q_nope must be"):
        ops.latent_attention_expanded(qn[..., :64], qr, kn, kr, v, cu, cu, SCALE)
    with pytest.raises(ValueError, match="k_nope must be"):
        ops.latent_attention_expanded(qn, qr, kn[:, :2], kr, v, cu, cu, SCALE)
    with pytest.raises(ValueError, match="v must be"):
        ops.latent_attention_expanded(qn, qr, kn, kr, v[:20], cu, cu, SCALE)
    with pytest.raises(ValueError, match="cu_q and cu_k"):
        ops.latent_attention_expanded(qn, qr, kn, kr, v, cu, i32([0, 20, 40]), SCALE)
    with pytest.raises(TypeError):
        ops.latent_attention_expanded(qn, qr, kn.float(), kr, v, cu, cu, SCALE)
    with pytest.raises(RuntimeError, match="code -2"):
        ops.latent_attention_expanded(qn, qr, kn, kr, v, cu, cu, 0.0)


@pytest.mark.parametrize("lens,new,H", [([5000], [3], 1), ([2100, 1500], [130, 7], 3), ([6000, 10], [20, 10], 2),
                                        ([1600, 0, 1700], [200, 0, 1], 4), ([1100, 1040], [1100, 2], 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_tokens_over_many_keys(ops, lens, new, H, causal):
    """The keys are cut into parts that are joined."""
    print(f"[case] expanded in parts lens={lens} new={new} H={H} causal={causal}", flush=True)
    assert ops.latent_attention_expanded_workspace_bytes(len(lens), sum(new), sum(lens), H) > 0
    c = Case(lens, new, H)
    c.check(*c.run(ops, causal=causal), causal=causal)


def test_parts_leave_padded_rows_and_replay(ops):
    print("[case] expanded in parts, padded, graph", flush=True)
    c = Case([2000, 1500], [60, 20], 4, spare=9)
    ws = torch.full((ops.latent_attention_expanded_workspace_bytes(2, 89, 3509, 4) // 4,), float("nan"), device="cuda")
    out = torch.full((89, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    _, lse = c.run(ops, out=out, workspace=ws)
    assert (out[80:] == 7).all()
    c.check(out, lse)
    args, cu_q, cu_k = c.tensors(), i32(starts(c.new)), i32(starts(c.lens))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.latent_attention_expanded(*args, cu_q, cu_k, SCALE)
    for new, lens in (([60, 20], [2000, 1500]), ([1, 70], [0, 3400]), ([80, 0], [500, 3000]), ([60, 20], [2000, 1500])):
        cu_q.copy_(i32(starts(new)))
        cu_k.copy_(i32(starts(lens)))
        g.replay()
        want = ops.latent_attention_expanded(*args, cu_q, cu_k, SCALE)
        torch.cuda.synchronize()
        assert torch.equal(got[:sum(new)], want[:sum(new)])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_parts_and_values_that_a_token_does_not_see(ops, value):
    print(f"[case] expanded in parts {value}", flush=True)
    c = Case([2100, 1400], [140, 40], 2)
    clean, _ = c.run(ops)
    c.v[1960 + 90, 1, 17] = value                 # new token 90's own key
    c.v[2100 + 5, 0, 3] = value                   # a key that all of the second sequence see
    out, _ = c.run(ops)
    got, want = out.float(), clean.float()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[90:140, 1, 17] = True
    hit[140:, 0, 3] = True
    assert torch.equal(got[~hit], want[~hit])
    if value != value:
        assert got[hit].isnan().all()
    else:
        assert (got[hit] == value).all()


@pytest.mark.parametrize("lens,new,H,causal", [
    ([300, 129, 64, 0, 257, 40], [129, 129, 64, 0, 200, 45], 96, True), ([200, 131], [200, 1], 256, True),
    ([90, 190, 70], [130, 60, 70], 192, False), ([(7 * i) % 61 for i in range(40)], [(5 * i) % 23 for i in range(40)], 24, True)])
def test_many_work_groups(ops, lens, new, H, causal):
    """Short tiles of many heads: two work-groups per CU."""
    print(f"[case] expanded {len(lens)} sequences, {H} heads, causal={causal}", flush=True)
    c = Case(lens, new, H)
    c.check(*c.run(ops, causal=causal), causal=causal)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_many_work_groups_and_values_that_a_token_does_not_see(ops, value):
    print(f"[case] expanded 160 heads {value}", flush=True)
    c = Case([250, 130], [240, 130], 160)
    clean, _ = c.run(ops)
    c.v[100, 101, 17] = value                     # new token 90
    c.v[250 + 129, 3, 64] = value                 # the last token's own
    out, _ = c.run(ops)
    got, want = out.float(), clean.float()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[90:240, 101, 17] = True
    hit[369, 3, 64] = True
    assert torch.equal(got[~hit], want[~hit])
    if value != value:
        assert got[hit].isnan().all()
    else:
        assert (got[hit] == value).all()
