"""Products with an epilogue at the ends of their range: infinite values through every activation, and the same bits of an
8-bit product, the sign of a zero included, at any number of rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import epilogue as o_epi

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("act", o_epi.ACTIVATIONS)
@pytest.mark.parametrize("m", [1, 40, 100, 700])
def test_infinite_values(nq, device, m, act):
    """Infinities from an operand, the bias, a scale and an overflowing sum, few rows and tiles: plus infinity stays, minus
    infinity is what the formula says."""

    from nari_qwen3_tts_amd.layers import linear_act, linear_int8

    n = 1030
    x, w = torch.zeros(m, 64, dtype=torch.bfloat16, device=device), torch.zeros(n, 64, dtype=torch.bfloat16, device=device)
    x[:, 0], w[:, 0] = 1.0, 1.0
    w[::2] *= -1.0
    bias = torch.zeros(n, dtype=torch.bfloat16, device=device)
    bias[5], bias[8] = INF, -INF
    x[m - 1, 0] = INF
    if m > 1:
        x[0, :4], w[:, 1:4] = 3e38, w[:, :1]  # sums beyond fp32
    with np.errstate(invalid="ignore", over="ignore"):
        y = (to_np(x).astype(np.float64) @ to_np(w).T.astype(np.float64)).astype(np.float32).astype(np.float64)
        want, bound = o_epi.product(y, to_np(bias), act), o_epi.bound(y, 0.0, to_np(bias), act)
    got = to_np(linear_act(x, w, bias, act)).astype(np.float64)
    assert np.isposinf(want).any() and (act in (None, "relu") or np.isnan(want).any())
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)])
    assert (np.abs(got[~odd] - want[~odd]) <= bound[~odd]).all()
    q, wq = torch.full((m, 64), 3, dtype=torch.int8, device=device), torch.full((n, 64), 5, dtype=torch.int8, device=device)
    wq[::2] *= -1
    s, sw = torch.ones(m, device=device), torch.full((n,), 1e-3, device=device)
    s[m - 1], sw[7], sw[10] = INF, INF, INF
    with np.errstate(invalid="ignore"):
        y = (to_np(q).astype(np.float64) @ to_np(wq).T.astype(np.float64)) * to_np(s)[:, None] * to_np(sw)
        want = o_epi.product(y, to_np(bias), act)
    got = to_np(linear_int8(q, s, wq, sw, bias=bias, activation=act)).astype(np.float64)
    odd = ~np.isfinite(want)
    assert np.isposinf(want).any()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)])


@pytest.mark.parametrize("act", o_epi.ACTIVATIONS)
@pytest.mark.parametrize("small", [False, True])
def test_int8_rows_have_the_same_bits_in_any_batch(nq, device, act, small):
    """Few-row kernels against tiles, with and without bias and residual; ``small``: products that leave zeros of either sign."""

    from nari_qwen3_tts_amd.layers import linear_int8

    rng = np.random.default_rng(5 + small)
    m, n, k = 300, 4100, 208
    q, w = (torch.from_numpy(rng.integers(-127, 128, (r, k)).astype(np.int8)).to(device) for r in (m, n))
    s, sw = (torch.from_numpy(rng.uniform(0.01, 0.1, r).astype(np.float32)).to(device) for r in (m, n))
    if small:
        s, sw = s * 1e-30, sw * 1e-30
    bias, res = (torch.from_numpy(rng.standard_normal(r).astype(np.float32)).to(device, torch.bfloat16) for r in ((n,), (m, n)))
    bias[::5] = -0.0
    res[:, ::3] = -0.0
    for b in (None, bias):
        for r in (None, res):
            out = linear_int8(q, s, w, sw, bias=b, activation=act, residual=r).view(torch.int16)
            assert not small or b is not None or r is not None or (out == -32768).any()
            for part in (slice(0, 1), slice(7, 23), slice(100, 140), slice(200, 264)):
                got = linear_int8(q[part], s[part], w, sw, bias=b, activation=act, residual=None if r is None else r[part])
                assert torch.equal(got.view(torch.int16), out[part])
