"""The draw by id among the kept tokens: the min-p sampler's oracle against closed forms and a walk (no GPU needed)."""

from __future__ import annotations

import numpy as np

from oracle import sampler as o_samp


def test_closed_forms():
    """A four-token row by hand: probabilities 4, 1, 8, 2 of 15 of the ids 0 to 3 at temperature 1."""

    x = np.log(np.array([4.0, 1.0, 8.0, 2.0]))

    def draw(u, k=0, p=1.0, m=0.0, t=1.0):
        return o_samp.sample_min_p_row(x, t, k, p, m, u, by_id=True)

    assert [draw(u) for u in (0.0, 0.26, 0.27, 0.33, 0.34, 0.86, 0.87, 1.0)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [draw(u, k=2) for u in (0.0, 0.33, 0.34, 1.0)] == [0, 0, 2, 2]  # ids 0 and 2, 4 and 8 of 12
    assert [draw(u, p=0.6) for u in (0.33, 0.34)] == [0, 2]  # 8 / 15 is short of it
    assert [draw(u, m=0.24) for u in (0.28, 0.29, 0.857, 0.858)] == [0, 2, 2, 3]  # 4, 8 and 2 of 14
    assert [draw(u, p=0.55, m=0.2) for u in (0.0, 1.0)] == [2, 2]  # 8 of 14 reach it
    assert [draw(u, t=0.0) for u in (0.0, 1.0)] == [2, 2]
    assert o_samp.sample_min_p([x] * 2, [1.0] * 2, [0] * 2, [1.0] * 2, [0.0] * 2, [0.2, 0.3]).tolist() == [0, 1]


def test_ties_at_the_cut_keep_the_lowest_ids():
    x = np.array([1.0, 0.0, 1.0, 1.0, 0.0])
    assert [o_samp.sample_min_p_row(x, 1.0, 2, 1.0, 0.0, u, by_id=True) for u in (0.0, 0.5, 0.51, 1.0)] == [0, 0, 2, 2]
    x[4] = 5.0  # the likeliest is the last id: of the ones the first alone is kept
    assert [o_samp.sample_min_p_row(x, 1.0, 2, 1.0, 0.0, u, by_id=True) for u in (0.0, 0.01, 0.02, 1.0)] == [0, 0, 4, 4]


def test_against_a_walk():
    """Tokens kept one by one in order of their logits, then walked by id, in float64, away from borders."""

    rng = np.random.default_rng(12)
    checked = 0
    for _ in range(300):
        v = int(rng.integers(1, 12))
        x, t, u = rng.standard_normal(v) * 2, float(np.float32(rng.uniform(0.3, 2))), float(np.float32(rng.random()))
        k, p, m = int(rng.integers(0, 8)), float(np.float32(rng.uniform(0.2, 1.1))), float(np.float32(rng.uniform(0, 0.5)))
        e = np.exp((x - x.max()) / t)
        ids = [i for i in sorted(range(v), key=lambda i: (-x[i], i))[: k or v] if e[i] >= m]
        kept, mass = [], 0.0
        for i in ids:
            if kept and mass >= p * e[ids].sum():
                break
            kept.append(i)
            mass += e[i]
        kept.sort()
        cum, by_rank = np.cumsum(e[kept]), np.cumsum(e[ids])
        if (np.abs(cum - u * cum[-1]) < 1e-9).any() or (np.abs(by_rank - p * by_rank[-1]) < 1e-9).any():
            continue
        checked += 1
        assert o_samp.sample_min_p_row(x, t, k, p, m, u, by_id=True) == kept[int(np.argmax(cum >= u * cum[-1]))]
    assert checked > 250
