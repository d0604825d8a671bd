"""GPU: the attention block at the edges of what its entry points take."""
import numpy as np
import pytest
import torch

from ferret_amd import lib
from oracle import attention as A
from tests.attention_helpers import SCALE, Batch, assert_near, bf16_tensor, bf16_values, i32, visible
from tests.test_gpu_expanded_attention import Case as Expanded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


@pytest.mark.parametrize("native", [True, False])
def test_expanded_rows_are_refused(ops, native, monkeypatch):
    """Many rows of one row's storage, which a row pitch cannot name; nothing is written."""
    print(f"[case] expanded rows, native={native}", flush=True)
    if not native:
        monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    rng = np.random.default_rng(1)
    x, w, r = (bf16_tensor(bf16_values(rng, *s)) for s in ((64, 512), (512,), (64, 64)))
    one, out = x[:1].expand(64, 512), torch.full((64, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.rms_norm(one, w, out=out), lambda: ops.rms_norm_e4m3(one, w)):
        with pytest.raises(ValueError, match="x's rows"):
            call()
    for call in (lambda: ops.rms_norm(x, w, one, out=out), lambda: ops.rms_norm_e4m3(x, w, one)):
        with pytest.raises(ValueError, match="residual's rows"):
            call()
    cache, table = ops.LatentCache.empty(4, 16), i32(range(4)).view(1, 4)
    with pytest.raises(ValueError, match="latent's rows"):
        ops.latent_cache_write(cache, one, r, table, i32([64]), i32([0, 64]))
    with pytest.raises(ValueError, match="rotary's rows"):
        ops.latent_cache_write(cache, x, r[:1].expand(64, 64), table, i32([64]), i32([0, 64]))
    torch.cuda.synchronize()
    assert (out == 7).all() and (cache.data == 0).all()
    # one row has any stride
    assert torch.equal(ops.rms_norm(x[0].expand(1, 512), w)[0], ops.rms_norm(x[:1], w)[0])


@pytest.mark.parametrize("H,n,length", [(16, 1, 200), (24, 1, 200), (128, 1, 200), (16, 1, 5000), (3, 4, 200), (4, 5, 200),
                                        (16, 5, 200), (1, 70, 200), (64, 3, 130), (16, 5, 5000)])
def test_an_infinite_latent_under_a_score_of_minus_infinity(ops, H, n, length):
    """bf16: such a key has no weight, and its Inf times that weight makes its column NaN for every token that
    sees it: in a step that all rows of a tile see and at the causal edge, alone and among other tokens."""
    print(f"[case] absorbed, Inf under -inf H={H} n={n} length={length}", flush=True)
    rng = np.random.default_rng(H + n)
    ql, qr = bf16_values(rng, n, H, 512), bf16_values(rng, n, H, 64)
    ql[..., 5] = -0.5
    for key in sorted({5, length - n, length - 2, length - 1}):
        b = Batch([length], 64, False, 41)
        table, lens = b.device()
        b.cache.data.view(-1, 576)[int(b.slots[0][key]), 5] = float("inf")
        out, lse = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32([0, n]), SCALE,
                                        return_lse=True)
        torch.cuda.synchronize()
        out, lse = out.float().cpu().numpy(), lse.cpu().numpy()
        see = visible(n, length)
        sees = see[:, key].copy()
        assert np.isnan(out[sees][..., 5]).all(), key
        see[:, key] = False
        k = np.concatenate([b.lat[0], b.rot[0]], 1)
        for h in range(H):
            o, ref, spread, reach = A.attend(np.concatenate([ql[:, h], qr[:, h]], 1), k, b.lat[0], SCALE, see)
            eo, el = A.bounds(o, ref, spread, reach, 576, length)
            got = out[:, h].copy()
            got[sees, 5] = o[sees, 5]
            assert_near(got, o, eo, f"key {key} head {h}")
            assert_near(lse[:, h], ref, el, f"lse key {key} head {h}")


@pytest.mark.parametrize("H,n", [(16, 1), (3, 4), (4, 5), (16, 5), (1, 70), (128, 1), (64, 3)])
@pytest.mark.parametrize("length", [200, 5000])
def test_a_key_without_weight_adds_nothing_whatever_its_scale(ops, H, n, length):
    """e4m3: a key that a token does not see, or whose term vanishes, counts as nothing, also where its latents
    stand 2^110 above those of the others."""
    print(f"[case] absorbed, scales 2^110 apart H={H} n={n} length={length}", flush=True)
    rng = np.random.default_rng(H + n)
    ql, qr = bf16_values(rng, n, H, 512), bf16_values(rng, n, H, 64)
    ql[...] = -np.abs(ql)
    k0 = Batch([length], 64, True, 43)
    table, lens = k0.device()
    want = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), k0.cache, table, lens, i32([0, n]), SCALE)
    hidden = length - 1 if n > 1 else None      # the last token's own key, which the others do not see
    for key in (hidden, 7):
        if key is None:
            continue
        b = Batch([length], 64, True, 43)
        row = int(b.slots[0][key])
        b.cache.data.view(-1, 640)[row, :512] = 0x38          # 1 in every column: the scores are below -2^110
        b.cache.scales.view(-1, 4)[row] = 247
        out, lse = ops.latent_attention(bf16_tensor(ql), bf16_tensor(qr), b.cache, table, lens, i32([0, n]), SCALE,
                                        return_lse=True)
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
        if key == hidden:
            assert torch.equal(out[:n - 1], want[:n - 1])
        out, lse = out.float().cpu().numpy(), lse.cpu().numpy()
        see = visible(n, length)
        see[:, key] = False
        k = np.concatenate([b.lat[0], b.rot[0]], 1)
        for h in range(H):
            o, ref, spread, reach = A.attend(np.concatenate([ql[:, h], qr[:, h]], 1), k, b.lat[0], SCALE, see)
            eo, el = A.bounds(o, ref, spread, reach, 576, length)
            assert_near(out[:, h], o, eo, f"key {key} head {h}")
            assert_near(lse[:, h], ref, el, f"lse key {key} head {h}")


@pytest.mark.parametrize("length,n,H", [(2000, 1, 1), (1200, 3, 1), (2700, 5, 3)])
def test_expanded_in_an_odd_number_of_parts_of_odd_rows(ops, length, n, H):
    print(f"[case] expanded in odd parts length={length} n={n} H={H}", flush=True)
    c = Expanded([length], [n], H)
    c.check(*c.run(ops))


@pytest.mark.parametrize("native", [True, False])
def test_overlapping_tensors_are_refused(ops, native, monkeypatch):
    print(f"[case] overlaps, native={native}", flush=True)
    if not native:
        monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    rng = np.random.default_rng(2)
    b = Batch([100, 30], 16, False, 1)
    (table, lens), cu = b.device(), i32([0, 1, 2])
    room = bf16_tensor(bf16_values(rng, 3, 4, 512))
    ql, qr = room[:2], bf16_tensor(bf16_values(rng, 2, 4, 64))
    before = b.cache.data.clone()
    ws = torch.empty(ops.latent_attention_workspace_bytes(2, 2, 4), dtype=torch.uint8, device="cuda")
    inside = b.cache.data.view(-1)[:100 * 576]
    for call in (lambda: ops.latent_attention(ql, qr, b.cache, table, lens, cu, SCALE, out=room[1:]),
                 lambda: ops.latent_attention(ql, qr, b.cache, table, lens, cu, SCALE, out=inside[:4096].view(2, 4, 512)),
                 lambda: ops.latent_attention(ql, qr, b.cache, table, lens, cu, SCALE, workspace=ws,
                                              out=ws[:8192].view(torch.bfloat16).view(2, 4, 512)),
                 lambda: ops.latent_cache_read(b.cache, table, i32([0, 20, 40]), 40, inside[:40 * 512].view(40, 512)),
                 lambda: ops.latent_cache_write(b.cache, inside.view(100, 576)[:2, :512], qr[:, 0].contiguous(), table, lens,
                                                cu)):
        with pytest.raises(RuntimeError, match="code -2"):
            call()
    torch.cuda.synchronize()
    assert torch.equal(b.cache.data.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("H,n,length", [(16, 1, 5000), (16, 40, 300), (128, 2, 3000), (3, 4, 70)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_absorbed_in_place(ops, H, n, length, e4m3):
    """The output on its queries, in whole tiles and in tiles that are cut and joined."""
    print(f"[case] absorbed in place H={H} n={n} length={length} e4m3={e4m3}", flush=True)
    rng = np.random.default_rng(3)
    b = Batch([length, n + 1], 64, e4m3, 5)
    ql, qr = (bf16_tensor(bf16_values(rng, 2 * n, H, w)) for w in (512, 64))
    args = (qr, b.cache, *b.device(), i32([0, n, 2 * n]), SCALE)
    want = ops.latent_attention(ql, *args)
    got = ops.latent_attention(ql, *args, out=ql)
    torch.cuda.synchronize()
    assert got.data_ptr() == ql.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("lens,new,H", [([300, 129], [200, 129], 4), ([5000], [3], 2), ([200, 131], [200, 1], 256)])
def test_expanded_in_place(ops, lens, new, H):
    print(f"[case] expanded in place lens={lens} new={new} H={H}", flush=True)
    c = Expanded(lens, new, H)
    qn, *rest = c.tensors()
    qn = qn.contiguous()
    cu_q, cu_k = i32(np.cumsum([0, *new])), i32(np.cumsum([0, *lens]))
    want = ops.latent_attention_expanded(qn, *rest, cu_q, cu_k, SCALE)
    got = ops.latent_attention_expanded(qn, *rest, cu_q, cu_k, SCALE, out=qn)
    torch.cuda.synchronize()
    assert got.data_ptr() == qn.data_ptr() and torch.equal(got, want)


def test_overlapping_sequences_past_32_bits_of_steps_are_left_out(ops):
    """Starts that do not ascend: 350 sequences over the same 64 tokens, 4.7e10 steps; nothing is written."""
    print("[case] absorbed, overlapping sequences", flush=True)
    B, T, H = 700, 64, 128
    cache = ops.LatentCache.empty(1, 1 << 20)
    table = torch.zeros((B, 16), dtype=torch.int32, device="cuda")
    out = torch.full((T, H, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    cu = i32([T * (b % 2) for b in range(B)] + [T])
    ws = torch.zeros(ops.latent_attention_workspace_bytes(B, T, H), dtype=torch.uint8, device="cuda")
    ops.latent_attention(torch.zeros_like(out), out[..., :64].contiguous(), cache, table, i32([1 << 24] * B), cu, SCALE,
                         out=out, workspace=ws)
    torch.cuda.synchronize()
    assert (out == 7).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_positions_far_below_zero_are_dropped(ops, e4m3):
    """lens - n + i below -2^31 is a negative position like any other."""
    print(f"[case] cache write far below zero e4m3={e4m3}", flush=True)
    c = ops.LatentCache.empty(3, 16, torch.float8_e4m3fn if e4m3 else torch.bfloat16)
    before = c.data.clone()
    x, r = (torch.ones((20, w), dtype=torch.bfloat16, device="cuda") for w in (512, 64))
    table = i32([0, 1, 2]).view(1, 3)
    for length, end in ((-2 ** 31, 2 ** 31 - 1), (-2 ** 31 + 5, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 20), (-1, 2 ** 31 - 1)):
        ops.latent_cache_write(c, x, r, table, i32([length]), i32([0, end]))
    torch.cuda.synchronize()
    assert torch.equal(c.data, before)
