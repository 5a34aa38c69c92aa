"""The min-p sampler's oracle against closed forms and brute force, and the entry point's refusals (no GPU needed)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sampler as o_samp


def test_min_p_row_closed_forms():
    """Cuts of a four-token row by hand: probabilities 8, 4, 2, 1 of 15 (ids 2, 0, 3, 1) at temperature 1."""

    x = np.log(np.array([4.0, 1.0, 8.0, 2.0]))

    def draw(u, k=0, p=1.0, m=0.0, t=1.0):
        return o_samp.sample_min_p_row(x, t, k, p, m, u)

    assert [draw(u) for u in (0.0, 0.5, 0.54, 0.79, 0.81, 0.93, 0.94, 1.0)] == [2, 2, 0, 0, 3, 3, 1, 1]
    assert [draw(u, k=2) for u in (0.6, 0.7, 1.0)] == [2, 0, 0]
    assert [draw(u, m=0.24) for u in (0.57, 0.58, 0.86, 1.0)] == [2, 0, 3, 3]  # of 8, 4, 2
    assert [draw(u, p=0.6) for u in (0.66, 0.67, 1.0)] == [2, 0, 0]  # 8 / 15 is short of it
    assert draw(1.0, p=0.55, m=0.2) == 2 and draw(1.0, p=0.55) == 0  # the share is of what min-p leaves: 8 of 14
    assert draw(1.0, p=0.0) == 2 and draw(1.0, m=1.0) == 2 and draw(0.99, t=0.0) == 2
    assert o_samp.sample_min_p_row(np.array([-np.inf, np.nan, -np.inf]), 1.0, 0, 1.0, 0.0, 0.9) == 0
    assert o_samp.sample_min_p_row(np.array([np.nan, 0.0, np.inf, np.inf]), 1.0, 0, 1.0, 0.0, 0.9) == 3


def test_min_p_row_against_brute_force():
    """A float64 restatement that keeps tokens one by one, away from borders."""

    rng = np.random.default_rng(11)
    for _ in range(300):
        v = int(rng.integers(1, 12))
        x, t, u = rng.standard_normal(v) * 2, float(np.float32(rng.uniform(0.3, 2))), float(np.float32(rng.random()))
        k, p, m = int(rng.integers(0, 8)), float(np.float32(rng.uniform(0.2, 1.1))), float(np.float32(rng.uniform(0, 0.5)))
        e = np.exp((x - x.max()) / t)
        ids = sorted(range(v), key=lambda i: (-x[i], i))[: k or v]
        ids = [i for i in ids if e[i] >= m]
        kept, mass = [], 0.0
        for i in ids:
            if kept and mass >= p * e[ids].sum():
                break
            kept.append(i)
            mass += e[i]
        cum = np.cumsum(e[kept])
        if (np.abs(cum - u * cum[-1]) < 1e-9).any() or (np.abs(cum - p * e[ids].sum()) < 1e-9).any():
            continue
        assert o_samp.sample_min_p_row(x, t, k, p, m, u) == kept[int(np.argmax(cum >= u * cum[-1]))]


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros(8)), ValueError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(logits=torch.zeros(8, 2).t()), ValueError),
    (dict(temperature=torch.ones(2, dtype=torch.float64)), TypeError),
    (dict(top_k=torch.ones(2, dtype=torch.int64)), TypeError),
    (dict(top_p=torch.ones(3)), ValueError),
    (dict(min_p=torch.ones(4)[::2]), ValueError),
    (dict(min_p=torch.ones(2, 1)), ValueError),
    (dict(uniforms=torch.ones(1).expand(2)), ValueError),
    (dict(out=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(out=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(), ValueError),  # the call itself, but on the CPU
])
def test_min_p_refusals(nq, change, error):
    from nari_qwen3_tts_amd.sampling import sample_min_p

    args = dict(logits=torch.zeros(2, 8), temperature=torch.ones(2), top_k=torch.zeros(2, dtype=torch.int32),
                top_p=torch.ones(2), min_p=torch.zeros(2), uniforms=torch.zeros(2))
    args.update(change)
    with pytest.raises(error):
        sample_min_p(**args)


def test_host_checks_of_the_min_p_entry(nq):
    """Refused before any launch (placeholder pointers)."""

    from nari_qwen3_tts_amd import _lib

    def call(logits=16, dtype=0, s0=64, rows=2, vocab=64, rest=(16, 16, 16, 16, 16, 16)):
        return _lib.load().nq_sample_min_p(logits, dtype, s0, rows, vocab, *rest, None)

    assert call(rows=0) == 0 and call(rows=-1) == -1 and call(vocab=0) == -1 and call(logits=None) == -1 and call(s0=-1) == -1
    for i in range(6):
        assert call(rest=[None if j == i else 16 for j in range(6)]) == -1
    assert call(vocab=(1 << 20) + 1) == -2 and call(dtype=2) == -2 and call(logits=2) == -2 and call(logits=1, dtype=1) == -2
