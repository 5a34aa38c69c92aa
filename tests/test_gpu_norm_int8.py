"""RMS norm answered in int8 codes and row scales against the float64 oracle: residuals and codes equal.  A scale is
max |p| / (127 sqrt(ss / K + eps)) with max |p| exact; a lane adds at most K / 64 squares and the lanes' sums take 10
more additions, of which the root halves the relative error, as it does the mean's and eps's; the root, the product
and the quotient round once each: (K / 64 + 12) / 2 + 3 roundings of 2^-24, and one for the square of the bound."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import int8 as o_int8

pytestmark = pytest.mark.gpu


def _bf16(rng, device, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(device, torch.bfloat16)


def _check(q, s, res, want):
    want_res, want_q, want_s = want
    assert res is None or np.array_equal(to_np(res), want_res, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), want_q)
    got = s.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want_s))
    keep = ~np.isnan(want_s)
    bound = ((q.shape[1] / 64 + 12) / 2 + 4) * 2.0**-24 * want_s + 2.0**-150  # subnormal scales: half of 2^-149
    assert (np.abs(got - want_s)[keep] <= bound[keep]).all(), np.abs(got / want_s - 1)[keep].max()


@pytest.mark.parametrize("width", [16, 48, 64, 512, 528, 1024, 1040, 2048, 2064, 4096, 6144, 8192, 8208, 20000])
@pytest.mark.parametrize("rows", [1, 2, 5, 67])
def test_add_norm(nq, device, rows, width):
    from nari_qwen3_tts_amd.layers import add_rmsnorm_int8

    rng = np.random.default_rng(rows * 31 + width)
    hidden, residual = _bf16(rng, device, rows, width), _bf16(rng, device, rows, width, std=4.0)
    weight = _bf16(rng, device, width)
    want = o_int8.add_rmsnorm(to_np(hidden), to_np(residual), to_np(weight), 1e-6)
    kept = hidden.clone()
    q, s = add_rmsnorm_int8(hidden, residual, weight, 1e-6)
    _check(q, s, residual, want)
    assert torch.equal(hidden, kept)


@pytest.mark.parametrize("rows,width", [(1, 16), (3, 1024), (9, 2048), (2, 9216), (700, 256), (3000, 2048)])
def test_norm(nq, device, rows, width):
    from nari_qwen3_tts_amd.layers import rmsnorm_int8

    rng = np.random.default_rng(rows + width)
    x, weight = _bf16(rng, device, rows, width), _bf16(rng, device, width)
    kept = x.clone()
    q, s = rmsnorm_int8(x, weight, 1e-5)
    _check(q, s, None, o_int8.add_rmsnorm(None, to_np(x), to_np(weight), 1e-5))
    assert torch.equal(x, kept)


@pytest.mark.parametrize("width", [64, 2064])
def test_extreme_rows(nq, device, width):
    """Zeros, NaN, infinities, sums that overflow bf16, values whose squares overflow or vanish, ties, no eps."""

    from nari_qwen3_tts_amd.layers import add_rmsnorm_int8, rmsnorm_int8

    rng = np.random.default_rng(width)
    x = _bf16(rng, device, 13, width)
    x[0] = 0
    x[1, 3], x[2, 5], x[3, width - 1] = float("nan"), float("inf"), float("-inf")
    x[4] *= 2.0**110
    x[5] *= 2.0**-120
    x[6] = 0
    x[6, 7] = 9.183549615799121e-41  # the smallest
    x[7] = 3.3895313892515355e38
    x[8, ::2] = 2.0**100
    x[9] = torch.arange(width, device=device) % 48 - 20.5  # quotients that tie
    x[10, 1:] = 0
    x[11] *= 2.0**62
    x[12] *= 2.0**-33
    for power in (0, 60, -70):
        weight = _bf16(rng, device, width, std=2.0**power)
        weight[9:20] = 2.0**power  # ties survive
        for eps in (0.0, 1e-6):
            q, s = rmsnorm_int8(x, weight, eps)
            _check(q, s, None, o_int8.add_rmsnorm(None, to_np(x), to_np(weight), eps))
    residual = x.clone()
    residual[7] = 3e38
    want = o_int8.add_rmsnorm(to_np(x), to_np(residual), to_np(weight), 1e-6)
    assert np.isinf(want[0][7]).all()
    _check(*add_rmsnorm_int8(x, residual, weight, 1e-6), residual, want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_weight_that_is_not_finite(nq, device, bad):
    from nari_qwen3_tts_amd.layers import rmsnorm_int8

    x, weight = torch.ones(3, 32, dtype=torch.bfloat16, device=device), torch.ones(32, dtype=torch.bfloat16, device=device)
    weight[31] = bad
    x[1, 31] = 0  # 0 times infinity
    q, s = rmsnorm_int8(x, weight, 1e-6)
    assert s.isnan().all() and not q.any()


def test_every_product(nq, device):
    """Codes of significands that are products of two, under a maximum that is one: against integer arithmetic."""

    from nari_qwen3_tts_amd.layers import rmsnorm_int8

    rng = np.random.default_rng(3)
    a, w = rng.integers(128, 256, (512, 4096)), rng.integers(128, 256, 4096)
    shift = rng.integers(0, 9, 4096)
    w_real = w * 2.0 ** -shift.astype(np.float64)
    p = (a * w) << (9 - shift)  # integers, in units of 2^-9
    top = p.max(1, keepdims=True)
    whole, rest = (254 * p) // (2 * top), (254 * p) % (2 * top)
    codes = whole + ((rest > top) | ((rest == top) & (whole % 2 == 1)))
    x, weight = (torch.from_numpy(t).to(device, torch.bfloat16) for t in (a.astype(np.float64), w_real))
    q, _ = rmsnorm_int8(x, weight, 1e-6)
    assert np.array_equal(q.cpu().numpy(), codes)


@pytest.mark.parametrize("width", [80, 2048, 2080])
def test_strided_rows(nq, device, width):
    """Rows as slices of wider ones, codes into a wider buffer; what lies beside them stays."""

    from nari_qwen3_tts_amd.layers import add_rmsnorm_int8, rmsnorm_int8

    rng = np.random.default_rng(width)
    h, r = (_bf16(rng, device, 6, width + 24)[:, 8:width + 8] for _ in range(2))
    wide = r._base if r._base is not None else r
    before = wide.clone()
    weight = _bf16(rng, device, width)
    want = o_int8.add_rmsnorm(to_np(h), to_np(r), to_np(weight), 1e-6)
    q = torch.full((6, width + 32), 99, dtype=torch.int8, device=device)
    s = torch.zeros(6, device=device)
    got = add_rmsnorm_int8(h, r, weight, 1e-6, q[:, 16:width + 16], s)
    assert got[1] is s
    _check(q[:, 16:width + 16], s, r, want)
    assert (q[:, :16] == 99).all() and (q[:, width + 16:] == 99).all()
    assert torch.equal(wide[:, :8], before[:, :8]) and torch.equal(wide[:, width + 8:], before[:, width + 8:])
    one = _bf16(rng, device, 1, width)
    q, s = rmsnorm_int8(one.expand(5, width), weight, 1e-6)  # one row read five times
    _check(q, s, None, o_int8.add_rmsnorm(None, np.repeat(to_np(one), 5, 0), to_np(weight), 1e-6))


def test_offsets_past_32_bits(nq, device):
    from nari_qwen3_tts_amd.layers import add_rmsnorm_int8

    rng = np.random.default_rng(6)
    big = torch.zeros(70, 1 << 26, dtype=torch.bfloat16, device=device)
    h, r = big[:, :128], big[:, 1 << 20:][:, :128]
    h.copy_(_bf16(rng, device, 70, 128))
    r.copy_(_bf16(rng, device, 70, 128))
    weight = _bf16(rng, device, 128)
    want = o_int8.add_rmsnorm(to_np(h), to_np(r), to_np(weight), 1e-6)
    _check(*add_rmsnorm_int8(h, r, weight, 1e-6), r, want)


def test_rows_do_not_depend_on_each_other(nq, device):
    """The same bits for a row alone and among others, on another stream, and captured; no rows at all."""

    from nari_qwen3_tts_amd.layers import add_rmsnorm_int8, rmsnorm_int8

    rng = np.random.default_rng(8)
    for rows, width in ((1500, 1024), (40, 6144)):
        x, h, weight = _bf16(rng, device, rows, width), _bf16(rng, device, rows, width), _bf16(rng, device, width)
        q, s = rmsnorm_int8(x, weight, 1e-6)
        q1, s1 = rmsnorm_int8(x[rows - 1:], weight, 1e-6)
        assert torch.equal(q[-1:], q1) and torch.equal(s[-1:], s1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q2, s2 = rmsnorm_int8(x, weight, 1e-6)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(q, q2) and torch.equal(s, s2)
        r = x.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            add_rmsnorm_int8(h, r, weight, 1e-6, q2, s2)
        for _ in range(3):
            r.copy_(_bf16(rng, device, rows, width))
            eager = r.clone()
            q, s = add_rmsnorm_int8(h, eager, weight, 1e-6)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(r, eager)
        q, s = add_rmsnorm_int8(h[:0], r[:0], weight, 1e-6)
        assert q.shape == (0, width) and s.shape == (0,)
