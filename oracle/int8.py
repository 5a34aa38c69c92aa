"""Oracle for the int8 row quantisation and product (test infrastructure only), in float64 and int64.

Pinned by tests/test_oracle_int8.py with closed forms and exact fractions.
"""

from __future__ import annotations

import numpy as np

from . import bf16


def quantize_rows(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Codes int8 rint(127 x / max |x|) and float64 scales max |x| / 127; a zero row has scale 1, a row with a
    NaN or an infinity codes of 0 and a NaN scale.  float64 holds 127 x and separates every quotient of bf16
    values from a tie that it is not."""

    x = np.asarray(x, dtype=np.float64)
    codes, scales = np.zeros(x.shape, np.int8), np.ones(x.shape[0])
    for r, row in enumerate(x):
        if not np.isfinite(row).all():
            scales[r] = np.nan
        elif np.abs(row).max() > 0:
            top = np.abs(row).max()
            codes[r], scales[r] = np.rint(127 * row / top), top / 127
    return codes, scales


def linear(q: np.ndarray, scales: np.ndarray, weight_q: np.ndarray, weight_scales: np.ndarray) -> np.ndarray:
    """float64 [M, N]; the integer sums are exact."""

    sums = q.astype(np.float64) @ weight_q.astype(np.float64).T  # below 2^53
    return sums * np.asarray(scales, np.float64)[:, None] * np.asarray(weight_scales, np.float64)


def add_rmsnorm(hidden: np.ndarray | None, residual: np.ndarray, weight: np.ndarray, eps: float):
    """(new residual, codes, float64 scales): the bf16 sum (the rows themselves without ``hidden``), and of its unrounded
    rmsnorm y the scales max |y| / 127 and the codes rint(127 p / max |p|), p = x * weight, whose quotients the
    division by the row's root leaves alone; zero, NaN and infinite rows as in ``quantize_rows``."""

    x = residual if hidden is None else bf16.round_f32((residual + hidden).astype(np.float32))
    p = np.asarray(x, np.float64) * np.asarray(weight, np.float64)  # 16 bits a product
    codes, scales = quantize_rows(p)
    fine = np.isfinite(scales) & (np.abs(np.where(np.isfinite(p), p, 0.0)).max(1) > 0)
    with np.errstate(invalid="ignore", over="ignore"):
        root = np.sqrt(np.mean(np.asarray(x, np.float64) ** 2, axis=1) + float(np.float32(eps)))
    scales[fine] = scales[fine] / root[fine]
    return x, codes, scales
