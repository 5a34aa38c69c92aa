"""The int8 oracle against closed forms and exact fractions, and the entry points' refusals (no GPU needed)."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import bf16 as o_bf16
from oracle import int8 as o_int8


def test_quantize_rows_closed_forms():
    x = np.array([[127.0, -1.0, 0.5, 1.5], [0, 0, 0, 0], [-2.0, 1.0, 2.0, 0.0], [np.nan, 1, 2, 3], [1, np.inf, 0, 0]])
    codes, scales = o_int8.quantize_rows(x)
    assert codes.tolist() == [[127, -1, 0, 2], [0] * 4, [-127, 64, 127, 0], [0] * 4, [0] * 4]  # 63.5 -> 64
    assert scales[:3].tolist() == [1.0, 1.0, 2 / 127] and np.isnan(scales[3:]).all()


def test_quantize_rows_against_fractions():
    x = o_bf16.round_f32(np.random.default_rng(1).standard_normal((20, 64)).astype(np.float32))
    codes, _ = o_int8.quantize_rows(x)
    for row, got in zip(x, codes):
        top = max(abs(Fraction(float(v))) for v in row)
        assert got.tolist() == [round(127 * Fraction(float(v)) / top) for v in row]  # round: ties to even


def test_quotients_keep_away_from_ties():
    """Every pair of bf16 significands and every exponent between them that matters: 127 a / (b 2^k) is a tie or at least
    1 / (254 a) > 2^-16 of itself from one, in integers; and float64 quotients round as the exact ones."""

    a, b = np.arange(1, 256)[:, None], np.arange(128, 256)[None, :]
    for k in range(12):
        num, den = 254 * a, b << k  # the quotient in halves
        if k == 0:
            a_max = np.minimum(a, b)
            num = 254 * a_max
        near = 2 * ((num // den) // 2) + 1  # the odd number of halves around it
        off = np.abs(num - near * den)
        assert (((off == 0) | (off * 254 * np.minimum(a, 255) >= num)).all()) and ((off == 0) | (off * 2**16 > num)).all()
        whole, rest = num // (2 * den), num % (2 * den)
        exact = whole + ((rest > den) | ((rest == den) & (whole % 2 == 1)))
        assert np.array_equal(np.rint(num / (2 * den)).astype(np.int64), exact)


def test_linear_closed_form():
    q, w = np.array([[1, 2], [-127, 127]], np.int8), np.array([[3, 4], [127, -127], [0, 1]], np.int8)
    y = o_int8.linear(q, [0.5, 2.0], w, [1.0, 1.0, 4.0])
    assert y.tolist() == [[5.5, -63.5, 4.0], [254.0, -64516.0, 1016.0]]


@pytest.mark.parametrize("x,q,scales,error", [
    (torch.zeros(2, 32), None, None, TypeError),
    (torch.zeros(2, 24, dtype=torch.bfloat16), None, None, ValueError),
    (torch.zeros(2, 0, dtype=torch.bfloat16), None, None, ValueError),
    (torch.zeros(32, dtype=torch.bfloat16), None, None, ValueError),
    (torch.zeros(32, 16, dtype=torch.bfloat16).t(), None, None, ValueError),
    (torch.zeros(2, 32, dtype=torch.bfloat16), torch.zeros(2, 32, dtype=torch.uint8), None, TypeError),
    (torch.zeros(2, 32, dtype=torch.bfloat16), torch.zeros(3, 32, dtype=torch.int8), None, ValueError),
    (torch.zeros(2, 32, dtype=torch.bfloat16), None, torch.zeros(3), ValueError),
    (torch.zeros(2, 32, dtype=torch.bfloat16), None, None, ValueError),  # the call itself, but on the CPU
])
def test_quantize_refusals(nq, x, q, scales, error):
    from nari_qwen3_tts_amd.layers import quantize_int8_rows

    with pytest.raises(error):
        quantize_int8_rows(x, q, scales)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 32)), TypeError),
    (dict(weight_q=torch.zeros(3, 32, dtype=torch.uint8)), TypeError),
    (dict(scales=torch.zeros(2, dtype=torch.float64)), TypeError),
    (dict(scales=torch.zeros(3)), ValueError),
    (dict(weight_scales=torch.zeros(6)[::2]), ValueError),
    (dict(weight_q=torch.zeros(3, 48, dtype=torch.int8)), ValueError),
    (dict(q=torch.zeros(2, 24, dtype=torch.int8), weight_q=torch.zeros(3, 24, dtype=torch.int8)), ValueError),
    (dict(q=torch.zeros(32, 2, dtype=torch.int8).t()), ValueError),
    (dict(out=torch.zeros(2, 3)), ValueError),
    (dict(out=torch.zeros(2, 4, dtype=torch.bfloat16)), ValueError),
    (dict(), ValueError),  # the call itself, but on the CPU
])
def test_linear_refusals(nq, change, error):
    from nari_qwen3_tts_amd.layers import linear_int8

    args = dict(q=torch.zeros(2, 32, dtype=torch.int8), scales=torch.zeros(2),
                weight_q=torch.zeros(3, 32, dtype=torch.int8), weight_scales=torch.zeros(3))
    args.update(change)
    with pytest.raises(error):
        linear_int8(**args)


def test_host_checks_of_the_c_entries(nq):
    """Refused before any launch (placeholder pointers)."""

    from nari_qwen3_tts_amd import _lib

    lib = _lib.load()

    def quantize(x=16, x_s0=64, m=2, k=64, q=16, q_s0=64, scales=16):
        return lib.nq_quantize_int8_rows(x, x_s0, m, k, q, q_s0, scales, None)

    assert quantize(m=0) == 0
    assert quantize(m=-1) == -1 and quantize(x=None) == -1 and quantize(k=0) == -1 and quantize(q_s0=32) == -1
    assert quantize(k=40, q_s0=40) == -2 and quantize(x=8) == -2 and quantize(x_s0=66) == -2 and quantize(q=4) == -2

    def linear(x=16, x_s0=64, w=16, w_s0=64, m=2, n=3, k=64, out=16, o_s0=3):
        return lib.nq_linear_int8(x, x_s0, 16, w, w_s0, 16, m, n, k, out, o_s0, None)

    assert linear(m=0) == 0 and linear(n=0) == 0
    assert linear(m=-1) == -1 and linear(x=None) == -1 and linear(k=0) == -1 and linear(o_s0=2) == -1
    assert linear(k=40) == -2 and linear(x=8) == -2 and linear(x_s0=72) == -2 and linear(w_s0=72) == -2
    assert linear(k=(1 << 17) + 16, x_s0=1 << 18, w_s0=1 << 18) == -2
