"""The attention block around the projections in 64 bits: norm, latent cache and latent
attention, from their formulas (numpy; test infrastructure only).

The reference computes none of these; the contracts are the library's own
(include/ferret_hip.h).
"""
from __future__ import annotations

import numpy as np

from oracle import formats as F

LATENT, ROTARY = 512, 64
MIN_BYTE = 16


def rms_norm(x: np.ndarray, w: np.ndarray, residual: np.ndarray | None, eps: float):
    """(y, s) in 64 bits for x, w, residual given as their values."""
    s = x.astype(np.float64) + (0.0 if residual is None else residual.astype(np.float64))
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    return y, s


def latent_quantize(x: np.ndarray):
    """Values [n, 512] -> (e4m3 codes uint8 [n, 512], exponent bytes uint8 [n, 4])."""
    n = x.shape[0]
    b = x.astype(np.float64).reshape(n, 4, 128)
    finite = np.where(np.isfinite(b), np.abs(b), 0.0)
    amax = finite.max(-1)
    # 448 = 0.875 * 2^9: the mantissa m in [0.5, 1) of amax needs one power more past 0.875
    m, e = np.frexp(amax)
    byte = np.where(amax > 0, e - 9 + (m > 0.875) + 127, MIN_BYTE).clip(min=MIN_BYTE).astype(np.int64)
    scaled = np.ldexp(b, (127 - byte)[..., None])
    bad = ~np.isfinite(scaled)
    codes = F.f32_to_e4m3(np.where(bad, 0.0, scaled).astype(np.float32))
    codes = np.where(bad, np.uint8(0x7F), codes)
    return codes.reshape(n, LATENT).astype(np.uint8), byte.astype(np.uint8)


def latent_dequantize(codes: np.ndarray, byte: np.ndarray) -> np.ndarray:
    v = F.e4m3_to_f32(codes).astype(np.float64).reshape(-1, 4, 128)
    return np.ldexp(v, (byte.astype(np.int64) - 127)[..., None]).reshape(-1, LATENT)


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float, visible: np.ndarray):
    """One sequence and head: q [n, d], k [m, d], v [m, e], visible [n, m] of truth values.

    Returns o [n, e], lse [n], spread [n, e] = sum_j p_j |v_j| and reach [n] =
    scale * max_j sum_d |q_d k_d|: the quantities that the rounding errors scale with.
    Rows that see nothing: zeros and -inf.
    """
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    n, m = q.shape[0], k.shape[0]
    if m == 0:
        z = np.zeros((n, v.shape[1]))
        return z, np.full(n, -np.inf), z, np.zeros(n)
    s = np.where(visible, (q @ k.T) * scale, -np.inf)
    top = s.max(-1)
    base = np.where(np.isfinite(top), top, 0.0)
    p = np.exp(s - base[:, None])
    total = p.sum(-1)
    some = total > 0
    p = p / np.where(some, total, 1.0)[:, None]
    with np.errstate(divide="ignore"):
        lse = np.where(some, base + np.log(np.where(some, total, 1.0)), -np.inf)
    reach = scale * np.where(visible, np.abs(q) @ np.abs(k).T, 0.0).max(-1)
    return p @ v, lse, p @ np.abs(v), reach


def bounds(o, lse, spread, reach, width: int, keys: int):
    """How far a kernel's (out in bf16, lse in fp32) may be off these values.

    fp32 sums of `width` exact products are off by at most width * 2^-24 of the sum of
    their magnitudes, so scores by reach * (width + 2) * 2^-24 (the scale's product and
    the subtraction of the maximum round too, to half a step of at most twice the
    reach), and exp2 by 2^-22 relative: a softmax term by `eta`, as numerator
    and through the sum, whose `keys` additions add keys * 2^-24 each.  A term
    is rounded to bf16, half a step is 2^-8 of it (spread), and so is the
    result (2^-8 of |o|).
    """
    eta = reach * (width + 6) * 2.0 ** -24 + 2.0 ** -22
    out = (2.0 ** -8 + 2 * eta[:, None] + 2 * (keys + 8) * 2.0 ** -24) * spread * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(o)
    level = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    return out, eta + (keys + 8) * 2.0 ** -24 + (level + 2) * 2.0 ** -22
