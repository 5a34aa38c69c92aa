"""Oracle for the paged K/V cache in 8 bits and the attention over it (test infrastructure only).

Restates in float64, apart from the kernels:

- the write: per run of tokens in consecutive slots of one block of 16, a power-of-two scale per kind and
  head, the least s >= 2^-126 with max |x| / s <= 127, grown to hold what the block has already; codes
  rint(x / s), earlier codes rint(code * old / new);
- attention over code * scale with the bottom-right causal rule of ``oracle.attention``, with bounds
  on what fp32 scores, a bf16 P and a bf16 output may lose.

Pinned by tests/test_oracle_kv_int8.py with closed forms.
"""

from __future__ import annotations

import numpy as np

BLOCK = 16
MIN_SCALE = 2.0**-126


def scale_for(amax: float) -> float:
    """The least power of two s >= 2^-126 with amax / s <= 127, by search from the exponent below it."""

    if amax == 0:
        return MIN_SCALE
    s = 2.0 ** (int(np.floor(np.log2(amax))) - 8)
    while amax > 127 * s:
        s *= 2
    return max(s, MIN_SCALE)


def write(codes: np.ndarray, scales: np.ndarray, key: np.ndarray, value: np.ndarray, pages, offsets) -> None:
    """In place: codes int8 [P, 2, ps, H, D], scales float32 [P, 2, ps // 16, H]; key, value [T, H, D]."""

    total, _, ps, heads, _ = codes.shape
    t, n = 0, len(pages)
    while t < n:
        p, o = int(pages[t]), int(offsets[t])
        if not (0 <= p < total and 0 <= o < ps):
            t += 1
            continue
        run = 1
        while (t + run < n and int(pages[t + run]) == p and int(offsets[t + run]) == o + run and (o + run) % BLOCK):
            run += 1
        b, first = o // BLOCK, o % BLOCK
        for kind, x in ((0, key), (1, value)):
            for h in range(heads):
                new = x[t : t + run, h].astype(np.float64)
                old = float(scales[p, kind, b, h]) if first else 0.0
                before = codes[p, kind, b * BLOCK : o, h].astype(np.float64)
                if not np.isfinite(new).all() or not 0 <= old < np.inf:
                    scales[p, kind, b, h] = np.nan
                    codes[p, kind, o : o + run, h] = 0
                    continue
                s = scale_for(float(np.abs(new).max()))
                if first:
                    s = max(s, old)
                codes[p, kind, b * BLOCK : o, h] = np.rint(before * (old / s)) if first else before
                codes[p, kind, o : o + run, h] = np.rint(new / s)
                scales[p, kind, b, h] = s
        t += run


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """code * scale, float64, [P, 2, ps, H, D]."""

    return codes.astype(np.float64) * np.repeat(scales.astype(np.float64), BLOCK, axis=2)[..., None]


def attention(q, codes, scales, kv_indptr, kv_indices, last_page_len, qo_indptr=None, sm_scale=None):
    """(out, bound) float64 [tokens, Hq, D]; tokens of no row are NaN in both.

    ``bound``: how far a kernel with fp32 scores, maxima and sums, P * v_scale rounded to bf16 and a bf16
    output may be off.  u = 2^-24.  A score is a sum of D exact products in fp32, each partial sum off by
    at most 2 u of sum |q k| (2: whatever the order and the rounding of the matrix unit), times two
    rounded factors, so its error is at most e = ((2 D + 4) u) sum |q k| sm_scale; subtracting the
    maximum in units of log2 adds 4 u max |s|, the exponential 4 u.  So P is off by a factor within
    2 e + 8 u max |s| + 8 u (the maximum's own error cancels between P and their sum), P * v_scale by a further
    2^-8, both against A = sum P |v| / l, the sums over n keys by 2 n u of the same, the output by 2^-8 of itself.
    """

    q = np.asarray(q, dtype=np.float64)
    tokens, hq, d = q.shape
    ps, hkv = codes.shape[2], codes.shape[3]
    g = hq // hkv
    scale = d**-0.5 if sm_scale is None else float(sm_scale)
    rows = len(kv_indptr) - 1
    qo = np.arange(rows + 1) if qo_indptr is None else np.asarray(qo_indptr)
    out = np.full(q.shape, np.nan)
    bound = np.full(q.shape, np.nan)
    u = 2.0**-24
    for r in range(rows):
        q0, q1 = int(qo[r]), int(qo[r + 1])
        ids = np.asarray(kv_indices[kv_indptr[r] : kv_indptr[r + 1]])
        kv_len = (len(ids) - 1) * ps + int(last_page_len[r]) if len(ids) else 0
        held = values(codes[ids], scales[ids]) if len(ids) else np.zeros((0, 2, ps, hkv, d))
        k = held[:, 0].reshape(-1, hkv, d)[:kv_len]
        v = held[:, 1].reshape(-1, hkv, d)[:kv_len]
        for i in range(q1 - q0):
            n = min(max(kv_len - (q1 - q0) + i + 1, 0), kv_len)
            for h in range(hq):
                if n == 0:
                    out[q0 + i, h] = bound[q0 + i, h] = 0.0
                    continue
                kh, vh, x = k[:n, h // g], v[:n, h // g], q[q0 + i, h]
                s = kh @ x * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                mean, size = p @ vh, p @ np.abs(vh)
                e = (2 * d + 4) * u * float((np.abs(kh) @ np.abs(x)).max()) * scale
                loss = 2 * e + 8 * u * float(np.abs(s).max()) + 8 * u + 2.0**-8 + 2 * n * u
                out[q0 + i, h] = mean
                bound[q0 + i, h] = 2.0**-8 * np.abs(mean) + loss * (1 + 2.0**-7) * size + 1e-38
    return out, bound


def attention_rows(q, codes, scales, kv_indptr, kv_indices, last_page_len, qo_indptr, num_pages=None):
    """``attention`` a row and head at a time, for rows of many queries; page ids outside [0, num_pages) have no
    keys.  The same bound (``num_pages``: how many pages the call was given, all by default)."""

    q = np.asarray(q, dtype=np.float64)
    tokens, hq, d = q.shape
    ps, hkv = codes.shape[2], codes.shape[3]
    pages = codes.shape[0] if num_pages is None else num_pages
    out, bound = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    u = 2.0**-24
    for r in range(len(kv_indptr) - 1):
        q0, q1 = int(qo_indptr[r]), int(qo_indptr[r + 1])
        ids = np.asarray(kv_indices[kv_indptr[r] : kv_indptr[r + 1]])
        kv_len = (len(ids) - 1) * ps + int(last_page_len[r]) if len(ids) else 0
        if kv_len == 0:
            out[q0:q1] = bound[q0:q1] = 0.0
            continue
        there = (ids >= 0) & (ids < pages)
        held = values(codes[np.where(there, ids, 0)], scales[np.where(there, ids, 0)])
        limit = np.clip(kv_len - (q1 - q0) + np.arange(q1 - q0) + 1, 0, kv_len)
        seen = (np.arange(kv_len) < limit[:, None]) & np.repeat(there, ps)[:kv_len]
        n = seen.sum(1, keepdims=True)
        for h in range(hq):
            k, v = (held[:, i, :, h // (hq // hkv)].reshape(-1, d)[:kv_len] for i in (0, 1))
            x = q[q0:q1, h]
            s = np.where(seen, x @ k.T * d**-0.5, -np.inf)
            top = np.where(n > 0, s.max(1, keepdims=True), 0.0)
            p = np.exp(s - top)
            p /= np.where(n > 0, p.sum(1, keepdims=True), 1.0)
            largest = np.where(seen, np.abs(x) @ np.abs(k).T, 0.0).max(1, keepdims=True) * d**-0.5
            size = np.where(seen, np.abs(x @ k.T) * d**-0.5, 0.0).max(1, keepdims=True)
            loss = 2 * (2 * d + 4) * u * largest + 8 * u * size + 8 * u + 2.0**-8 + 2 * n * u
            out[q0:q1, h] = p @ v
            bound[q0:q1, h] = np.where(n > 0, 2.0**-8 * np.abs(p @ v) + loss * (1 + 2.0**-7) * (p @ np.abs(v)) + 1e-38, 0.0)
    return out, bound
