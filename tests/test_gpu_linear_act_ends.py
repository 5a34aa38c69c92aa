"""Products with an epilogue at the ends of their range: infinite values through every activation."""

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
