"""Batches for the latent cache and attention tests, built on the host with the oracle's quantizer."""
from __future__ import annotations

import numpy as np
import torch

from ferret_amd import ops
from oracle import attention as A
from oracle import formats as F

SCALE = 192.0 ** -0.5


def bf16_values(rng, *shape, std=1.0):
    return F.bf16_round((rng.standard_normal(shape) * std).astype(np.float32))


def bf16_tensor(x: np.ndarray) -> torch.Tensor:
    """bf16 values (as float32, possibly Inf or NaN) -> a tensor on the GPU."""
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).cuda()


def i32(v) -> torch.Tensor:
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def starts(counts) -> list[int]:
    return [0, *np.cumsum(counts).tolist()]


class Batch:
    """Sequences in a paged cache: shuffled pages, garbage (NaN where `poison`) in every slot that no key has."""

    def __init__(self, lens, page, e4m3, seed, extra_pages=2, poison=False, spare_columns=0):
        rng = np.random.default_rng(seed)
        self.lens, self.page, self.e4m3 = list(lens), page, e4m3
        per = [-(-n // page) for n in lens]
        self.pages = sum(per) + extra_pages
        order = rng.permutation(self.pages)
        self.table = np.full((len(per), max([1, *per]) + spare_columns), -1, dtype=np.int32)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        lat = [bf16_values(rng, n, 512) * np.exp2(rng.integers(-2, 3, 512)).astype(np.float32) for n in lens]
        rot = [bf16_values(rng, n, 64) for n in lens]
        self.rot = [r.astype(np.float64) for r in rot]
        rows = self.pages * page
        junk = np.full if poison else (lambda shape, _: bf16_values(rng, *shape, std=3.0))
        lat_pool, rot_pool = junk((rows, 512), np.nan), junk((rows, 64), np.nan)
        self.slots = [self.slots_of(b, n) for b, n in enumerate(lens)]
        for s, x, r in zip(self.slots, lat, rot):
            lat_pool[s], rot_pool[s] = x, r
        if e4m3:
            codes, byte = A.latent_quantize(lat_pool)
            if poison:
                byte[:] = 255
                for s, x in zip(self.slots, lat):
                    byte[s] = A.latent_quantize(x)[1]
            self.lat = [A.latent_dequantize(codes[s], byte[s]) for s in self.slots]
            data = np.concatenate([codes, F.f32_to_bf16_bits(rot_pool.astype(np.float32)).view(np.uint8)], 1)
            self.cache = ops.LatentCache(torch.from_numpy(data).cuda().view(self.pages, page, 640),
                                         torch.from_numpy(byte).cuda().view(self.pages, page, 4))
        else:
            self.lat = [x.astype(np.float64) for x in lat]
            self.cache = ops.LatentCache(bf16_tensor(np.concatenate([lat_pool, rot_pool], 1)).view(
                self.pages, page, 576))

    def slots_of(self, b, n):
        pos = np.arange(n)
        return self.table[b, pos // self.page].astype(np.int64) * self.page + pos % self.page

    def device(self):
        return torch.from_numpy(self.table).cuda(), i32(self.lens)


def visible(n, length, causal=True):
    """[n, length]: what token i of n new ones sees of `length` keys."""
    if not causal:
        return np.ones((n, length), dtype=bool)
    return np.arange(length)[None] <= (length - n + np.arange(n))[:, None]


def assert_near(got: np.ndarray, want: np.ndarray, bound: np.ndarray, what: str):
    assert np.array_equal(np.isfinite(got), np.isfinite(want)), f"{what}: Inf or NaN differ"
    fine = np.isfinite(want)
    off = np.abs(got[fine].astype(np.float64) - want[fine])
    worst = float((off / (bound[fine] + 1e-30)).max()) if off.size else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"
    return worst


def check_absorbed(batch: Batch, new, ql, qr, out, lse, causal=True, scale=SCALE, what=""):
    """out [T, H, 512] and lse [T, H] against the oracle on the values ql [T, H, 512], qr [T, H, 64]."""
    out, lse = out.float().cpu().numpy(), lse.cpu().numpy()
    t, worst = 0, 0.0
    for b, (length, n) in enumerate(zip(batch.lens, new)):
        k = np.concatenate([batch.lat[b], batch.rot[b]], 1)
        see = visible(n, length, causal)
        for h in range(ql.shape[1]):
            q = np.concatenate([ql[t:t + n, h], qr[t:t + n, h]], 1)
            o, ref, spread, reach = A.attend(q, k, batch.lat[b], scale, see)
            eo, el = A.bounds(o, ref, spread, reach, 576, length)
            worst = max(worst, assert_near(out[t:t + n, h], o, eo, f"{what} seq {b} head {h}"))
            assert_near(lse[t:t + n, h], ref, el, f"{what} lse seq {b} head {h}")
        t += n
    return worst
