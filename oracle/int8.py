"""Oracle for the int8 row quantisation and product (test infrastructure only), in float64 and int64.

Pinned by tests/test_oracle_int8.py with closed forms and exact fractions.
"""

from __future__ import annotations

import numpy as np


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
