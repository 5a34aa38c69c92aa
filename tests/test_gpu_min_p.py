"""Min-p sampling against the oracle: tokens equal.  The weights are integers of 2^-42 from a double exponential; an
ulp of it, 2^-53, moves a weight by at most one unit now and then, and a sum by a share of some 2^-40, so that a
uniform of 24 bits lands between the two sums about once in 2^20 draws at the largest vocabularies."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import sampler as o_samp

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _vec(device, values, dtype=torch.float32):
    return torch.tensor(values, dtype=dtype, device=device)


def _run(device, logits, temperature, top_k, top_p, min_p, u):
    """The tokens, checked against the oracle's; parameters as lists, one entry a row."""

    from nari_qwen3_tts_amd.sampling import sample_min_p

    got = sample_min_p(logits, _vec(device, temperature), _vec(device, top_k, torch.int32), _vec(device, top_p),
                       _vec(device, min_p), _vec(device, u)).cpu().numpy()
    want = o_samp.sample_min_p(to_np(logits), temperature, top_k, top_p, min_p, u)
    bad = np.nonzero(got != want)[0]
    assert not len(bad), [(r, got[r], want[r], temperature[r], top_k[r], top_p[r], min_p[r], u[r]) for r in bad[:5]]
    return got


def _logits(rng, device, rows, vocab, dtype, std=2.0):
    x = rng.standard_normal((rows, vocab)) * std
    x += (rng.random((rows, vocab)) < min(0.25, 40 / vocab)) * rng.uniform(2, 8, (rows, vocab))
    return torch.from_numpy(x.astype(np.float32)).to(device, dtype)


def _uniforms(rng, n):
    return [float(v) for v in rng.integers(0, 1 << 24, n) / np.float32(1 << 24)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 3, 8, 63, 64, 65, 257, 1000, 2048, 4096, 4097, 8191, 20000, 65537])
def test_tokens(nq, device, vocab, dtype):
    """Every kind of row: wide and narrow cuts, each alone and together, decided and flat logits."""

    rng = np.random.default_rng(vocab)
    cuts = [(t, k, p, m) for t in (0.0, 0.7, 1.0, 3.0) for k in (0, 1, 5, 50, 700, 5000) for p in (1.0, 0.9, 0.3)
            for m in (0.0, 0.05, 0.5)]
    if vocab > 8192:
        cuts = [cuts[i] for i in rng.permutation(len(cuts))[:64]]
    t, k, p, m = (list(v) for v in zip(*cuts))
    for std in (2.0, 0.25):
        _run(device, _logits(rng, device, len(cuts), vocab, dtype, std), t, k, p, m, _uniforms(rng, len(cuts)))


@pytest.mark.parametrize("vocab", [151936, 262144, 1 << 20])
def test_large_vocabularies(nq, device, vocab):
    rng = np.random.default_rng(vocab)
    cuts = [(1.0, 0, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1), (1.3, 50, 0.9, 0.0), (1.0, 20000, 0.7, 0.0),
            (0.0, 0, 1.0, 0.0), (2.0, 0, 0.99, 0.001), (9.0, 100000, 0.5, 0.0)]
    t, k, p, m = (list(v) for v in zip(*cuts))
    for dtype in (torch.bfloat16, torch.float32):
        _run(device, _logits(rng, device, len(cuts), vocab, dtype), t, k, p, m, _uniforms(rng, len(cuts)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 4096, 4100, 70000])
def test_ties(nq, device, vocab, dtype):
    """Logits all equal, and of two or three values: ranks are ids, down to the last digit of an id."""

    rng = np.random.default_rng(vocab + 1)
    x = torch.full((12, vocab), -3.25, dtype=dtype, device=device)
    x[4:8] += torch.from_numpy(rng.integers(0, 2, (4, vocab))).to(device)
    x[8:] += torch.from_numpy(rng.integers(0, 3, (4, vocab)) * 0.5).to(device)
    for k, p, m in ((0, 1.0, 0.0), (vocab // 2 + 1, 1.0, 0.0), (0, 0.5, 0.0), (vocab - 1, 0.75, 0.7), (1, 0.5, 1.0)):
        _run(device, x, [1.0] * 12, [k] * 12, [p] * 12, [m] * 12, _uniforms(rng, 12))
    # equal weights: u = (r + 1/2) / V draws rank r, and u = (r + 1) / V still does
    r = rng.integers(0, 4096, 12)
    flat = torch.zeros(12, 4096, dtype=dtype, device=device)
    assert np.array_equal(_run(device, flat, [1.0] * 12, [0] * 12, [1.0] * 12, [0.0] * 12, [(v + 0.5) / 4096 for v in r]), r)
    assert np.array_equal(_run(device, flat, [1.0] * 12, [0] * 12, [1.0] * 12, [0.0] * 12, [(v + 1.0) / 4096 for v in r]), r)
    # top-p of half of them keeps half of them
    assert np.array_equal(_run(device, flat, [1.0] * 12, [0] * 12, [0.5] * 12, [0.0] * 12, [1.0] * 12), [2047] * 12)


@pytest.mark.parametrize("vocab", [70, 5003])
def test_masked_and_infinite_logits(nq, device, vocab):
    rng = np.random.default_rng(vocab)
    x = _logits(rng, device, 16, vocab, torch.float32)
    x[0] = -INF
    x[1] = NAN
    x[2, 1:] = -INF
    x[3, :-1] = -INF
    x[4, ::2] = -INF
    x[5, 1::2] = NAN
    x[6, 33] = INF
    x[7, 10:60] = INF
    x[8] = torch.finfo(torch.float32).min
    x[9, ::3] = torch.finfo(torch.float32).min
    x[10] = torch.finfo(torch.float32).max
    x[11, 7], x[11, 9] = 0.0, -0.0
    x[11, :7] = x[11, 10:] = -1e-30
    x[11, 8] = -0.0
    x[12] *= 1e30
    x[13] *= 1e-30
    x[14, :] = NAN
    x[14, 5] = 2.0
    x[15, 3], x[15, 4] = INF, NAN
    for t in (1.0, 0.0, INF, 1e-30, 1e-45, 1e30, -1.0, NAN):
        for k, p, m in ((0, 1.0, 0.0), (3, 1.0, 0.0), (0, 0.6, 0.0), (0, 1.0, 0.2), (40, 0.9, 0.01)):
            got = _run(device, x, [t] * 16, [k] * 16, [p] * 16, [m] * 16, _uniforms(rng, 16))
            assert (got[:2] == 0).all() and got[2] == 0 and got[3] == vocab - 1 and got[6] == 33 and 10 <= got[7] < 60
            assert got[14] == 5 and got[15] == 3
            _run(device, x.to(torch.bfloat16), [t] * 16, [k] * 16, [p] * 16, [m] * 16, _uniforms(rng, 16))


@pytest.mark.parametrize("vocab", [65, 3000, 9001])
def test_every_kind_of_nan(nq, device, vocab):
    """Quiet and signalling NaN of both signs, in the first places and the last, are never the maximum."""

    rng = np.random.default_rng(vocab)
    x = _logits(rng, device, 12, vocab, torch.bfloat16, 1.0)
    bits = x.view(torch.int16)
    for i, nan in enumerate((0x7f81, 0x7fff, 0x7fc0, -0x7f, -1, -0x40)):
        bits[i, ::2], bits[i + 6, 1::2] = nan, nan
        bits[i, -1] = bits[i + 6, 0] = nan
    assert (x.isnan().sum(1) >= vocab // 2).all()
    for t, m in ((1.0, 0.0), (1.0, 0.05), (0.0, 0.0)):
        got = _run(device, x, [t] * 12, [0, 20] * 6, [0.9, 1.0, 1.0] * 4, [m] * 12, _uniforms(rng, 12))
        assert not x.cpu()[torch.arange(12), torch.from_numpy(got)].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [1.0, 2.0**-20, 2.0**20, 2.0**-110])
def test_small_and_zero_logits(nq, device, dtype, scale):
    """Rows whose logits are far apart in size: zeros of either sign, values 40 binades and more below the largest, the
    smallest ones; and some that are too far below the maximum to count, or are none."""

    rng = np.random.default_rng(3)
    rows, vocab = 12, 9003
    x = torch.from_numpy((rng.standard_normal((rows, vocab)) * np.exp2(rng.integers(-60, 2, (rows, vocab)))).astype(np.float32))
    x[:, ::5] = 0.0
    x[:, 1::10] = -0.0
    x[:, 3::50] = 2.0**-125
    x[:, 7::70] = -1000.0
    x[:, 9::90] = -INF
    x[:, 11::110] = NAN
    x[6:, 100:8000] = 0.0
    x[9] = x[9].clamp(max=0.0)
    x = (x * scale).to(device, dtype)
    temperature = [float(np.float32(scale * t)) for t in (0.05, 0.3, 1.0, 3.0)] * 3
    for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (3000, 1.0, 0.0), (0, 0.95, 0.2)):
        _run(device, x, temperature, [k] * rows, [p] * rows, [m] * rows, _uniforms(rng, rows))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_greedy_ties_take_the_lowest_id(nq, device, dtype):
    """Maxima in the first and last places, which rows at odd addresses load alone, and between them."""

    vocab = 20011
    wide = torch.zeros(24, vocab + 7, dtype=dtype, device=device)
    for at in range(7):
        x = wide[:, at:at + vocab]
        x.fill_(-1.0)
        want = np.zeros(24, np.int64)
        for r in range(24):
            ids = [vocab - 1 - r % 3, vocab // 2 + 37 * r, 8191 + r, 8 + r] + ([r % 9] if r % 2 else [])
            x[r, ids] = 0.0
            if r % 4 == 0:
                x[r, ids[-1]] = -0.0
            want[r] = min(ids)
        assert np.array_equal(_run(device, x, [0.0] * 24, [0] * 24, [1.0] * 24, [0.0] * 24, [0.5] * 24), want)
        _run(device, x, [1.0] * 24, [3] * 24, [1.0] * 24, [0.0, 0.99] * 12, [0.9] * 24)


def test_large_offsets_beside_a_small_temperature(nq, device):
    """Where a bound on the logits that count is looser than the weights' range: those are counted and weigh nothing."""

    rng = np.random.default_rng(12)
    x = torch.from_numpy((1e6 + rng.random((12, 9000)) * 8).astype(np.float32)).to(device)
    for t in (1e-3, 0.01, 0.3):
        for k, p, m in ((0, 1.0, 0.0), (8500, 1.0, 0.0), (4000, 0.9, 0.0), (300, 1.0, 0.0), (0, 0.9, 0.1)):
            _run(device, x, [t] * 12, [k] * 12, [p] * 12, [m] * 12, _uniforms(rng, 12))
            _run(device, -x, [t] * 12, [k] * 12, [p] * 12, [m] * 12, _uniforms(rng, 12))


def test_parameters_out_of_range(nq, device):
    rng = np.random.default_rng(9)
    for vocab in (300, 9000):
        x = _logits(rng, device, 8, vocab, torch.bfloat16, 0.5)
        u = [0.0, 1.0, -1.0, 2.0, NAN, INF, -INF, 1 - 2.0**-24]
        for p, m, k in ((0.0, 0.0, 0), (-1.0, 0.0, 0), (NAN, NAN, -5), (2.0, -1.0, 1 << 30), (1.0, 1.0, 0), (INF, 7.0, 0),
                        (0.9, INF, 9)):
            _run(device, x, [1.0] * 8, [k] * 8, [p] * 8, [m] * 8, u)


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 1001), (torch.float32, 6007)])
def test_strides_streams_and_graphs(nq, device, dtype, vocab):
    """Rows at odd addresses, one row for all, another stream, replays with new inputs; a row alone and among others."""

    from nari_qwen3_tts_amd.sampling import sample_min_p

    rng = np.random.default_rng(vocab)
    wide = _logits(rng, device, 40, vocab + 9, dtype)
    t, k, p, m = [0.9] * 40, [0, 30] * 20, [0.95, 1.0] * 20, [0.0, 0.02, 0.0, 0.1] * 10
    u = _uniforms(rng, 40)
    for at in (0, 1, 5):
        x = wide[:, at:at + vocab]
        got = _run(device, x, t, k, p, m, u)
        alone = _run(device, x[17:18], t[17:18], k[17:18], p[17:18], m[17:18], u[17:18])
        assert alone[0] == got[17]
    _run(device, wide[:1, :vocab].expand(40, vocab), t, k, p, m, u)
    args = [_vec(device, t), _vec(device, k, torch.int32), _vec(device, p), _vec(device, m), _vec(device, u)]
    out = torch.full((42,), -7, dtype=torch.long, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert sample_min_p(x, *args, out=out[1:41]).data_ptr() == out[1:].data_ptr()
    torch.cuda.current_stream().wait_stream(side)
    assert np.array_equal(out[1:41].cpu().numpy(), got) and out[0] == -7 and out[41] == -7
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_min_p(x, *args, out=out[1:41])
    for _ in range(3):
        x.copy_(_logits(rng, device, 40, vocab, dtype))
        want = sample_min_p(x, *args)
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[1:41], want)
    assert sample_min_p(x[:0], *(a[:0] for a in args)).shape == (0,)


def test_offsets_past_32_bits(nq, device):
    rng = np.random.default_rng(4)
    big = torch.zeros(40, 1 << 26, dtype=torch.float32, device=device)
    x = big[:, 3:5003]
    x.copy_(_logits(rng, device, 40, 5000, torch.float32))
    _run(device, x, [1.0] * 40, [0] * 40, [0.9] * 40, [0.0, 0.05] * 20, _uniforms(rng, 40))


def test_frequencies(nq, device):
    """Equally spaced uniforms draw each kept token in proportion to its probability, and no other."""

    x = torch.tensor([2.0, 1.0, 0.0, -1.0, 1.5, -8.0], device=device)
    n = 1 << 14
    u = [(i + 0.5) / n for i in range(n)]
    got = _run(device, x.expand(n, 6), [0.8] * n, [4] * n, [0.97] * n, [0.04] * n, u)
    e = np.exp((x.cpu().numpy().astype(np.float64) - 2.0) / 0.8)
    e[[3, 5]] = 0  # min-p drops ids 3 and 5; of the rest top-p keeps what reaches 0.97
    assert e[[0, 4, 1]].sum() < 0.97 * e.sum()
    counts = np.bincount(got, minlength=6)
    assert (np.abs(counts - n * e / e.sum()) <= 1).all()
