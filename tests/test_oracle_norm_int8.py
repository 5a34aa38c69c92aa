"""The int8 norm's oracle against exact fractions, and the entry points' refusals (no GPU needed)."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import bf16 as o_bf16
from oracle import int8 as o_int8


def test_add_rmsnorm_against_fractions():
    """Codes of the unrounded norm in exact fractions; a row of zeros, one with an infinity; without eps the scale of
    a constant row is 1 / 127 of its weight."""

    rng = np.random.default_rng(2)
    x, h, w = (o_bf16.round_f32(rng.standard_normal((6, 32)).astype(np.float32)) for _ in range(3))
    w = w[0]
    x[4], h[4], x[5, 3] = 0, 0, np.inf
    res, codes, scales = o_int8.add_rmsnorm(h, x, w, 1e-6)
    assert np.array_equal(res, o_bf16.round_f32(x + h))
    for r in range(4):
        p = [Fraction(float(v)) * Fraction(float(u)) for v, u in zip(res[r], w)]
        top = max(abs(v) for v in p)
        assert codes[r].tolist() == [round(127 * v / top) for v in p]
        y = res[r].astype(np.float64) * w / np.sqrt(np.mean(res[r].astype(np.float64) ** 2) + 1e-6)
        assert abs(scales[r] - np.abs(y).max() / 127) <= 1e-12 * scales[r]
    assert not codes[4:].any() and scales[4] == 1 and np.isnan(scales[5])
    _, codes, scales = o_int8.add_rmsnorm(None, np.full((1, 16), -3.0, np.float32), np.full(16, 2.0, np.float32), 0.0)
    assert (codes == -127).all() and scales[0] == 2 / 127


@pytest.mark.parametrize("change,error", [
    (dict(residual=torch.zeros(2, 32)), TypeError),
    (dict(weight=torch.zeros(32)), TypeError),
    (dict(hidden=torch.zeros(2, 32)), TypeError),
    (dict(hidden=torch.zeros(3, 32, dtype=torch.bfloat16)), ValueError),
    (dict(hidden=torch.zeros(32, 2, dtype=torch.bfloat16).t()), ValueError),
    (dict(residual=torch.zeros(2, 2, 32, dtype=torch.bfloat16)), ValueError),
    (dict(hidden=torch.zeros(2, 24, dtype=torch.bfloat16), residual=torch.zeros(2, 24, dtype=torch.bfloat16),
          weight=torch.zeros(24, dtype=torch.bfloat16)), ValueError),
    (dict(weight=torch.zeros(48, dtype=torch.bfloat16)), ValueError),
    (dict(weight=torch.zeros(64, dtype=torch.bfloat16)[::2]), ValueError),
    (dict(eps=-1e-6), ValueError),
    (dict(eps=float("nan")), ValueError),
    (dict(q=torch.zeros(2, 32)), TypeError),
    (dict(q=torch.zeros(3, 32, dtype=torch.int8)), ValueError),
    (dict(scales=torch.zeros(2, dtype=torch.float64)), TypeError),
    (dict(scales=torch.zeros(3)), ValueError),
    (dict(), ValueError),  # the call itself, but on the CPU
])
def test_norm_refusals(nq, change, error):
    from nari_qwen3_tts_amd.layers import add_rmsnorm_int8, rmsnorm_int8

    args = dict(hidden=torch.zeros(2, 32, dtype=torch.bfloat16), residual=torch.zeros(2, 32, dtype=torch.bfloat16),
                weight=torch.zeros(32, dtype=torch.bfloat16), eps=1e-6)
    args.update(change)
    with pytest.raises(error):
        add_rmsnorm_int8(**args)
    if "hidden" not in change:
        args["hidden"] = args.pop("residual")
        with pytest.raises(error):
            rmsnorm_int8(**args)


def test_norm_refuses_its_own_residual(nq):
    from nari_qwen3_tts_amd.layers import add_rmsnorm_int8

    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="distinct"):
        add_rmsnorm_int8(x, x, torch.zeros(32, dtype=torch.bfloat16), 1e-6)


def test_host_checks_of_the_norm_entries(nq):
    """Refused before any launch (placeholder pointers)."""

    from nari_qwen3_tts_amd import _lib

    lib = _lib.load()

    def add(h=16, h_s0=64, r=16, r_s0=64, w=16, m=2, k=64, eps=0.0, q=16, q_s0=64, scales=16):
        return lib.nq_add_rmsnorm_int8(h, h_s0, r, r_s0, w, m, k, eps, q, q_s0, scales, None)

    assert add(m=0) == 0
    for bad in (dict(m=-1), dict(h=None), dict(r=None), dict(w=None), dict(k=0), dict(eps=-1.0), dict(eps=float("nan")),
                dict(q=None), dict(q_s0=32), dict(r_s0=32), dict(scales=None), dict(h_s0=-64)):
        assert add(**bad) == -1, bad
    for bad in (dict(k=40), dict(h=8), dict(r=8), dict(w=8), dict(q=4), dict(scales=2), dict(h_s0=66), dict(r_s0=66),
                dict(q_s0=68)):
        assert add(**bad) == -2, bad

    def norm(x=16, x_s0=64, m=2, k=64):
        return lib.nq_rmsnorm_int8(x, x_s0, 16, m, k, 0.0, 16, 64, 16, None)

    assert norm(m=0) == 0 and norm(x=None) == -1 and norm(x_s0=-8) == -1 and norm(x_s0=66) == -2 and norm(x=8) == -2
