"""The min-p sampler draws among the kept tokens by id: every way that a row can take, against the oracle and against
what the definition says directly.  Tokens are equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_min_p import _logits, _run, _uniforms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [7, 64, 300, 1500, 2049, 6001, 8192, 8193, 20011, 66000])
def test_every_way(nq, device, vocab, dtype):
    """Few, some and many kept tokens by each cut and by several; uniforms at both ends besides."""

    rng = np.random.default_rng(vocab)
    cuts = [(t, k, p, m) for t in (0.7, 1.3) for k in (0, 3, 200, 600, 5000) for p in (1.0, 0.95, 0.5)
            for m in (0.0, 0.001, 0.02, 0.3)]
    if vocab > 9000:
        cuts = [cuts[i] for i in rng.permutation(len(cuts))[:48]]
    t, k, p, m = (list(v) for v in zip(*cuts))
    for std in (1.0, 2.5):
        x = _logits(rng, device, len(cuts), vocab, dtype, std)
        _run(device, x, t, k, p, m, _uniforms(rng, len(cuts)))
        for u in (0.0, 1.0):
            _run(device, x, t, k, p, m, [u] * len(cuts))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 500, 1999, 5003, 9001, 30011])
def test_two_values(nq, device, vocab, dtype):
    """Every second id at 0, the others far below: of n ids the draw is the ceil(u n)-th, whatever the address."""

    n = (vocab + 1) // 2
    if n > 4096:
        n = 4000  # at most as many equal logits
    wide = torch.full((8, vocab + 8), -60.0, dtype=dtype, device=device)
    rank = np.array([0, 1, n // 3, n // 2, n - 2, n - 1, 5, n - 9])
    u = [float(np.float32((r + 0.5) / n)) for r in rank]
    for at in (0, 1, 3, 7):
        x = wide[:, at:at + vocab]
        x.fill_(-60.0)
        x[:, vocab - 2 * n + (vocab % 2)::2] = 0.0
        first = vocab - 2 * n + (vocab % 2)
        got = _run(device, x, [1.0] * 8, [0, vocab - 1] * 4, [1.0] * 8, [0.0, 0.0, 0.5, 0.5] * 2, u)
        assert np.array_equal(got, first + 2 * rank)


@pytest.mark.parametrize("vocab", [2000, 7000, 20000])
def test_the_order_of_the_logits_does_not_matter(nq, device, vocab):
    """A permutation of equal weights draws the same id; a kept set moved to other ids is walked in their order."""

    rng = np.random.default_rng(vocab)
    ids = np.sort(rng.permutation(vocab)[:300])
    values = np.linspace(1.0, 1.25, 300).astype(np.float32)
    x = np.full((8, vocab), -50.0, np.float32)
    for r in range(8):
        x[r, ids] = rng.permutation(values)
    u = _uniforms(rng, 8)
    for k, p, m in ((0, 1.0, 0.0), (300, 1.0, 0.0), (0, 1.0, 0.5), (250, 0.9, 0.0)):
        got = _run(device, torch.from_numpy(x).to(device), [1.0] * 8, [k] * 8, [p] * 8, [m] * 8, u)
        assert np.isin(got, ids).all()
        if p == 1.0 and k != 250:
            want = [ids[np.argmax(np.cumsum(np.exp(x[r, ids].astype(np.float64))) >=
                                  u[r] * np.exp(x[r, ids].astype(np.float64)).sum())] for r in range(8)]
            assert np.array_equal(got, want)


@pytest.mark.parametrize("vocab", [8192, 9001, 70001, 1 << 20])
@pytest.mark.parametrize("kind", ["equal", "neighbours", "hot", "two scales"])
def test_bins_that_overflow_the_list(nq, device, vocab, kind):
    """More logits in the cut's bin than the list holds, which the digits of logits and ids cut one to five times: the
    same tokens at each call, and the oracle's."""

    from nari_qwen3_tts_amd.sampling import sample_min_p

    rows = 4 if vocab > 100000 else 32
    rng = np.random.default_rng(vocab)
    x = np.full((rows, vocab), 1.5, np.float32)
    t = 1.0
    if kind == "neighbours":  # three values that differ in their last digits
        x = x + rng.integers(0, 3, x.shape).astype(np.float32) * np.float32(2.0**-23)
    elif kind == "hot":  # all of a bell within few bins
        x, t = rng.standard_normal(x.shape).astype(np.float32), 500.0
    elif kind == "two scales":  # equal ones below some that are not
        x[:, ::7] = rng.standard_normal((rows, len(range(0, vocab, 7)))) * 0.001 + 1.75
    x = torch.from_numpy(x).to(device)
    for k, p, m in ((vocab // 2, 1.0, 0.0), (0, 0.6, 0.0), (vocab - 9, 0.3, 0.0), (vocab // 3, 0.5, 0.2)):
        u = _uniforms(rng, rows)
        want = _run(device, x, [t] * rows, [k] * rows, [p] * rows, [m] * rows, u)
        args = [torch.tensor([v] * rows, device=device) for v in (t, k, p, m)] + [torch.tensor(u, device=device)]
        args[1] = args[1].int()
        for _ in range(8):
            assert np.array_equal(sample_min_p(x, *(a if a.dtype == torch.int32 else a.float() for a in args)).cpu().numpy(), want)


@pytest.mark.parametrize("vocab", [8192, 20480])
def test_the_last_kept_id(nq, device, vocab):
    """u = 1 asks for the whole mass: the passes that sum a row have to agree to the last unit.  Logits one below the
    largest, where a rounding of the exponent moves a weight of 2^-42 most often."""

    rows = 256
    rng = np.random.default_rng(vocab)
    x = (-1.0 - rng.random((rows, vocab)) * 0.1).astype(np.float32)
    x[:, 3] = 0.0
    x = torch.from_numpy(x).to(device)
    got = _run(device, x, [1.0] * rows, [0] * rows, [1.0] * rows, [0.0] * rows, [1.0] * rows)
    assert (got == vocab - 1).all()
    for temperature in (0.9, 1.1):
        _run(device, x, [temperature] * rows, [0, vocab // 2] * (rows // 2), [1.0, 1.0, 0.75, 0.5] * (rows // 4),
             [0.0] * rows, [1.0] * rows)
