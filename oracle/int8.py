"""The int8 quantizer and product as include/ferret_hip.h states them, in whole numbers and 64 bits."""
from __future__ import annotations

import numpy as np

from oracle import formats as F

LEAST = 2.0 ** -100


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """bf16 values [M, K] -> (int8 codes, fp32 scales): round(127 x / a), ties to even, a / 127.

    Decided in whole numbers: with x = X 2^e and a = A 2^f (8-bit X and A) a quotient is a
    ratio of integers, whose float64 quotient is exact at every half and at least 2^-18 from one elsewhere."""
    x = np.asarray(x, dtype=np.float64)
    bad = ~np.isfinite(x).all(axis=1)
    a = np.maximum(np.abs(np.where(np.isfinite(x), x, 0.0)).max(axis=1), LEAST)
    q = np.rint(np.where(np.isfinite(x), x, 0.0) * 127.0 / a[:, None]).astype(np.int8)
    q[bad] = 0
    scale = (a.astype(np.float32) / np.float32(127)).astype(np.float32)
    scale[bad] = np.nan
    return q, scale


def product(a: np.ndarray, sa: np.ndarray, b: np.ndarray, sb: np.ndarray, residual: np.ndarray | None = None):
    """The bf16 bits of (a . b^T) * sa * sb (+ residual): the sum exact, each later step rounded to fp32."""
    # float64 holds every sum exactly: |sum| <= 2^14 K < 2^53
    total = (a.astype(np.float64) @ b.astype(np.float64).T).astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        y = total * sa.astype(np.float32)[:, None] * sb.astype(np.float32)[None, :]
        if residual is not None:
            y = y + residual.astype(np.float32)
    return F.f32_to_bf16_bits(y.astype(np.float32))
