"""GPU: writing the paged latent cache and reading it back, bit for bit against the oracle's quantizer."""
import numpy as np
import pytest
import torch

from oracle import attention as A
from oracle import formats as F
from tests.attention_helpers import Batch, bf16_tensor, bf16_values, i32, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _pool(cache):
    data = _bytes(cache.data).reshape(cache.num_pages * cache.page_size, -1).copy()
    return data, None if cache.scales is None else _bytes(cache.scales).reshape(data.shape[0], 4).copy()


def _put(data, scales, slots, lat, rot):
    rot = F.f32_to_bf16_bits(rot.astype(np.float32)).view(np.uint8)
    if scales is None:
        data[slots] = np.concatenate([F.f32_to_bf16_bits(lat.astype(np.float32)).view(np.uint8), rot], 1)
    else:
        codes, byte = A.latent_quantize(lat)
        data[slots], scales[slots] = np.concatenate([codes, rot], 1), byte


BATCHES = [([1], [1]), ([16], [16]), ([5, 64, 33], [2, 1, 33]), ([130, 7, 0, 200], [100, 0, 0, 3]),
           ([3] * 70 + [40], [1] * 70 + [17])]


@pytest.mark.parametrize("lens,new", BATCHES)
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("e4m3", [False, True])
def test_write_then_read(ops, lens, new, page, e4m3):
    print(f"[case] cache write lens={lens[:4]} new={new[:4]} page={page} e4m3={e4m3}", flush=True)
    b = Batch(lens, page, e4m3, 5)
    table, dlens = b.device()
    rng = np.random.default_rng(1)
    T = sum(new)
    wide = bf16_values(rng, T + 3, 704)         # rows behind the last sequence, in a slice of a wider tensor
    wide[:, 64:] *= np.exp2(rng.integers(-20, 20, (T + 3, 1)))
    x = bf16_tensor(wide)
    data, scales = _pool(b.cache)
    ops.latent_cache_write(b.cache, x[:, 64:576], x[:, 640:], table, dlens, i32(starts(new)))
    t = 0
    for i, (length, n) in enumerate(zip(lens, new)):
        at = b.slots[i][length - n:]
        _put(data, scales, at, wide[t:t + n, 64:576], wide[t:t + n, 640:])
        t += n
    torch.cuda.synchronize()
    assert np.array_equal(_bytes(b.cache.data).reshape(data.shape), data)
    if e4m3:
        assert np.array_equal(_bytes(b.cache.scales).reshape(scales.shape), scales)
    # read everything back, more rows asked for than there are keys
    S = sum(lens)
    lat = torch.full((S + 5, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    rot = torch.full((S + 5, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.latent_cache_read(b.cache, table, i32(starts(lens)), S + 5, lat, rot)
    torch.cuda.synchronize()
    slots = np.concatenate([s for s in b.slots]) if S else np.zeros(0, np.int64)
    if e4m3:
        want = A.latent_dequantize(data[slots, :512], scales[slots])
        rows = data[slots][:, 512:].copy().view(np.uint16)
    else:
        want = F.bf16_bits_to_f32(data[slots][:, :1024].copy().view(np.uint16))
        rows = data[slots][:, 1024:].copy().view(np.uint16)
    assert np.array_equal(lat[:S].float().cpu().numpy().astype(np.float64), want)
    assert np.array_equal(rot[:S].float().cpu().numpy(), F.bf16_bits_to_f32(rows).reshape(S, 64))
    assert (lat[S:] == 7).all() and (rot[S:] == 7).all()


def test_quantizer_at_its_borders(ops):
    """Maxima on both sides of 448 * 2^k, every midpoint of the codes, zeros, subnormals, the largest bf16, Inf, NaN."""
    print("[case] cache quantizer borders", flush=True)
    rows = []
    for k in (-120, -60, -7, 0, 5, 100):
        for top in (448.0, 450.0, 446.0, 256.0, 255.0, 232.0):
            v = np.zeros(128, np.float32)
            grid = F.e4m3_to_f32(np.arange(0x00, 0x7F, dtype=np.uint8)).astype(np.float64)
            mids = np.concatenate([grid, (grid[1:] + grid[:-1]) / 2])
            pick = mids[mids <= 224][np.random.default_rng(k + 200).integers(0, (mids <= 224).sum(), 127)]
            v[:127], v[127] = np.ldexp(pick, k), np.ldexp(top, k)
            rows.append(F.bf16_round(v) * np.where(np.arange(128) % 2, 1, -1))
    rows += [np.zeros(128), np.full(128, 2.0 ** -133), np.full(128, F.bf16_round(np.float32(3.3e38)))]
    x = np.asarray(rows, dtype=np.float32)
    bad = np.tile(x[3], (3, 1))
    bad[0, 3], bad[1, 5], bad[2, :] = np.inf, np.nan, -np.inf
    x = np.concatenate([x, bad])
    x = np.concatenate([x, np.zeros((-len(x) % 4, 128), np.float32)]).reshape(-1, 512)
    T = len(x)
    c = ops.LatentCache.empty(2, 64, torch.float8_e4m3fn)
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    ops.latent_cache_write(c, bf16_tensor(x), bf16_tensor(np.zeros((T, 64))), table, i32([T]), i32([0, T]))
    torch.cuda.synchronize()
    codes, byte = A.latent_quantize(x)
    got = c.data[1, :T, :512].cpu().numpy()
    nan = (codes & 0x7F) == 0x7F
    assert np.array_equal((got & 0x7F) == 0x7F, nan)
    assert np.array_equal(got[~nan], codes[~nan]) and np.array_equal(c.scales[1, :T].cpu().numpy(), byte)


def test_what_is_no_page_is_left_alone(ops):
    """Entries outside the cache, positions before 0 and past the table, rows behind the last sequence."""
    print("[case] cache bad entries", flush=True)
    for e4m3 in (False, True):
        c = ops.LatentCache.empty(3, 16, torch.float8_e4m3fn if e4m3 else torch.bfloat16)
        c.data.fill_(1)
        before = _bytes(c.data).copy()
        table = torch.tensor([[-1, 3, 2 ** 31 - 1], [-2 ** 31, -1, 7]], dtype=torch.int32, device="cuda")
        x, r = bf16_tensor(np.ones((40, 512))), bf16_tensor(np.ones((40, 64)))
        ops.latent_cache_write(c, x, r, table, i32([48, 10]), i32([0, 20, 40]))       # 20 tokens, 10 positions
        ops.latent_cache_write(c, x, r, table, i32([2 ** 31 - 1, -5]), i32([0, 20, 40]))
        lat, rot = ops.latent_cache_read(c, table, i32([0, 30, 64]), 64)
        torch.cuda.synchronize()
        assert np.array_equal(_bytes(c.data), before)
        assert (lat == 0).all() and (rot == 0).all()


def test_offsets_past_32_bits(ops):
    """A page more than 4 GB into the cache."""
    print("[case] cache of 5 GB", flush=True)
    for dtype, width in ((torch.bfloat16, 1152), (torch.float8_e4m3fn, 640)):
        pages = 5 * 2 ** 30 // (64 * width)
        c = ops.LatentCache.empty(pages, 64, dtype)
        rng = np.random.default_rng(2)
        x, r = bf16_tensor(bf16_values(rng, 70, 512)), bf16_tensor(bf16_values(rng, 70, 64))
        table = torch.tensor([[pages - 1, 4]], dtype=torch.int32, device="cuda")
        ops.latent_cache_write(c, x, r, table, i32([70]), i32([0, 70]))
        lat, rot = ops.latent_cache_read(c, table, i32([0, 70]), 70)
        torch.cuda.synchronize()
        assert torch.equal(rot, r) and (c.data[pages - 2].float() == 0).all()
        if dtype == torch.bfloat16:
            assert torch.equal(lat, x)
        else:
            codes, byte = A.latent_quantize(x.float().cpu().numpy())
            assert np.array_equal(lat.double().cpu().numpy(), A.latent_dequantize(codes, byte))
        del c, lat, rot
        torch.cuda.empty_cache()


def test_refusals(ops):
    b = Batch([20, 30], 16, True, 1)
    table, lens = b.device()
    x, r, cu = bf16_tensor(np.ones((4, 512))), bf16_tensor(np.ones((4, 64))), i32([0, 2, 4])
    with pytest.raises(TypeError, match="LatentCache"):
        ops.latent_cache_write((b.cache.data, b.cache.scales), x, r, table, lens, cu)
    with pytest.raises(TypeError):
        ops.latent_cache_write(ops.LatentCache(b.cache.data), x, r, table, lens, cu)            # bytes without scales
    with pytest.raises(ValueError, match="cache.scales"):
        ops.latent_cache_write(ops.LatentCache(b.cache.data, b.cache.scales[:, :8].contiguous()), x, r, table, lens, cu)
    with pytest.raises(ValueError, match="640"):
        ops.latent_cache_write(ops.LatentCache(b.cache.data[..., :576].contiguous(), b.cache.scales), x, r, table,
                               lens, cu)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.latent_cache_read(ops.LatentCache(torch.zeros((2, 8, 576), dtype=torch.bfloat16, device="cuda")), table,
                              cu, 4)
    with pytest.raises(ValueError, match="page_table"):
        ops.latent_cache_write(b.cache, x, r, table, lens, i32([0, 4]))
    with pytest.raises(TypeError):
        ops.latent_cache_write(b.cache, x, r, table.long(), lens, cu)
    with pytest.raises(ValueError, match="rotary"):
        ops.latent_cache_write(b.cache, x, r[:3], table, lens, cu)
    with pytest.raises(ValueError, match="lens"):
        ops.latent_cache_write(b.cache, x, r, table, lens[:1], cu)
    with pytest.raises(ValueError, match="latent must have shape"):
        ops.latent_cache_read(b.cache, table, cu, 4, latent=x[:3])
    with pytest.raises(ValueError, match="bf16 or e4m3"):
        ops.LatentCache.empty(2, 16, torch.float16)
