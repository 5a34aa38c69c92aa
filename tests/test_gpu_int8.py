"""int8 row quantisation and product against the float64 oracle: codes equal; the sums are exact, so a product is
within its roundings, two of fp32 and one of bf16."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import int8 as o_int8

pytestmark = pytest.mark.gpu


def _bf16(rng, device, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(device, torch.bfloat16)


@pytest.mark.parametrize("rows,k", [(1, 16), (3, 48), (64, 2048), (5, 6144), (2, 8192), (3, 8208), (2, 20000), (300, 128)])
def test_quantize_rows(nq, device, rows, k):
    from nari_qwen3_tts_amd.layers import quantize_int8_rows

    x = _bf16(np.random.default_rng(rows + k), device, rows, k)
    q, s = quantize_int8_rows(x)
    want_q, want_s = o_int8.quantize_rows(to_np(x))
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert (np.abs(s.cpu().numpy() - want_s) <= 2.0**-24 * want_s).all()


def test_quantize_rows_extremes(nq, device):
    """Rows of zeros, of the smallest and largest values, of ties, of NaN and infinities; a strided input."""

    from nari_qwen3_tts_amd.layers import quantize_int8_rows

    buf = torch.zeros(9, 72, dtype=torch.bfloat16, device=device)
    x = buf[:, 8:56]
    x[1, 3] = 9.183549615799121e-41
    x[2, :3] = torch.tensor([3.3895313892515355e38, -1.6947656946257677e38, 1e-38])
    x[3] = torch.arange(48) - 20.5
    x[4, 7], x[5, 7], x[6, 47] = float("nan"), float("inf"), float("-inf")
    x[7, 1:9] = torch.tensor([2.0, 1.0, -1.0, 0.5, 1e-30, -2.0, 1.984375, 0.0078125])
    x[8] = 1e30
    q = torch.full((9, 64), 99, dtype=torch.int8, device=device)
    s = torch.zeros(9, device=device)
    quantize_int8_rows(x, q[:, 16:], s)
    want_q, want_s = o_int8.quantize_rows(to_np(x))
    assert np.array_equal(q[:, 16:].cpu().numpy(), want_q) and (q[:, :16] == 99).all()
    got = s.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want_s))
    keep = ~np.isnan(want_s)
    assert (np.abs(got - want_s)[keep] <= np.maximum(2.0**-24 * want_s[keep], 2.0**-150)).all()  # subnormal: half of 2^-149


def _codes(rng, device, rows, k):
    return torch.from_numpy(rng.integers(-127, 128, (rows, k)).astype(np.int8)).to(device)


def _check(out, q, s, w, sw):
    """bf16 (2^-8) of two fp32 roundings behind the integer's own (3 * 2^-24)."""

    want = o_int8.linear(*(t.cpu().numpy() for t in (q, s, w, sw)))
    bound = (2.0**-8 + 4 * 2.0**-24) * np.abs(want)
    got = to_np(out).astype(np.float64)
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


@pytest.mark.parametrize("n,k", [(16, 16), (1, 2048), (50, 144), (257, 1040), (1024, 2048), (130, 6144), (2048, 128)])
@pytest.mark.parametrize("m", [1, 2, 16, 17, 33, 64, 65, 100, 129, 300])
def test_linear(nq, device, m, n, k):
    from nari_qwen3_tts_amd.layers import linear_int8

    rng = np.random.default_rng(m * 7 + n + k)
    q, w = _codes(rng, device, m, k), _codes(rng, device, n, k)
    s = torch.from_numpy(rng.uniform(0.001, 2.0, m).astype(np.float32)).to(device)
    sw = torch.from_numpy(rng.uniform(0.001, 2.0, n).astype(np.float32)).to(device)
    out = linear_int8(q, s, w, sw)
    _check(out, q, s, w, sw)
    assert torch.equal(out[-1], linear_int8(q[-1:], s[-1:], w, sw)[0])  # the same bits at any number of rows


@pytest.mark.parametrize("m,n,k", [(2300, 2048, 256), (640, 6000, 528), (4000, 1111, 160)])
def test_linear_large(nq, device, m, n, k):
    from nari_qwen3_tts_amd.layers import linear_int8

    rng = np.random.default_rng(m)
    q, w = _codes(rng, device, m, k), _codes(rng, device, n, k)
    s, sw = torch.rand(m, device=device) + 0.01, torch.rand(n, device=device) + 0.01
    _check(linear_int8(q, s, w, sw), q, s, w, sw)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_linear_strided(nq, device, m):
    """Codes as slices of wider rows, an output whose rows are odd and whose neighbours stay."""

    from nari_qwen3_tts_amd.layers import linear_int8

    rng = np.random.default_rng(m)
    q, w = _codes(rng, device, m, 288)[:, 16:256], _codes(rng, device, 77, 272)[:, 32:]
    s, sw = torch.rand(m, device=device), torch.rand(77, device=device)
    out = torch.full((m, 83), 7.0, dtype=torch.bfloat16, device=device)
    linear_int8(q, s, w, sw, out=out[:, 3:80])
    _check(out[:, 3:80], q, s, w, sw)
    assert (out[:, :3] == 7.0).all() and (out[:, 80:] == 7.0).all()


@pytest.mark.parametrize("m", [1, 64, 200])
def test_linear_largest_sums(nq, device, m):
    """Every product 127 * 127 over the longest K the product takes: 2^31 is not reached."""

    from nari_qwen3_tts_amd.layers import linear_int8

    k = 1 << 17
    q = torch.full((m, k), 127, dtype=torch.int8, device=device)
    w = torch.full((20, k), -127, dtype=torch.int8, device=device)
    s, sw = torch.ones(m, device=device), torch.ones(20, device=device)
    _check(linear_int8(q, s, w, sw), q, s, w, sw)


def test_linear_empty_and_nan_rows(nq, device):
    from nari_qwen3_tts_amd.layers import linear_int8, quantize_int8_rows

    rng = np.random.default_rng(5)
    w, sw = quantize_int8_rows(_bf16(rng, device, 30, 64))
    x = _bf16(rng, device, 70, 64)
    x[4, 5], x[66, 0] = float("nan"), float("inf")
    x[9] = 0
    q, s = quantize_int8_rows(x)
    out = linear_int8(q, s, w, sw)
    assert out[4].isnan().all() and out[66].isnan().all() and not out[9].any()
    keep = [r for r in range(70) if r not in (4, 66)]
    _check(out[keep], q[keep], s[keep], w, sw)
    assert linear_int8(q[:0], s[:0], w, sw).shape == (0, 30)
    assert quantize_int8_rows(x[:0])[0].shape == (0, 64)


def test_linear_offsets_past_32_bits(nq, device):
    """Rows of x, weight rows and output rows that begin past 2^32 bytes or elements."""

    from nari_qwen3_tts_amd.layers import linear_int8

    rng = np.random.default_rng(6)
    big = torch.zeros(70, 1 << 26, dtype=torch.int8, device=device)
    q, w = big[:, :128], big[:, 1 << 20 :][:, :128]
    q.copy_(_codes(rng, device, 70, 128))
    w.copy_(_codes(rng, device, 70, 128))
    s, sw = torch.rand(70, device=device), torch.rand(70, device=device)
    out = torch.zeros(70, 1 << 26, dtype=torch.bfloat16, device=device)[:, :70]
    for rows in (70, 64):
        linear_int8(q[:rows], s[:rows], w, sw, out=out[:rows])
        _check(out[:rows], q[:rows], s[:rows], w, sw)


def test_graph(nq, device):
    from nari_qwen3_tts_amd.layers import linear_int8, quantize_int8_rows

    rng = np.random.default_rng(7)
    for m in (8, 300):
        x, out = _bf16(rng, device, m, 512), torch.zeros(m, 96, dtype=torch.bfloat16, device=device)
        w, sw = quantize_int8_rows(_bf16(rng, device, 96, 512))
        q, s = torch.empty(m, 512, dtype=torch.int8, device=device), torch.empty(m, device=device)
        linear_int8(*quantize_int8_rows(x, q, s), w, sw, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            linear_int8(*quantize_int8_rows(x, q, s), w, sw, out=out)
        for _ in range(3):
            x.copy_(_bf16(rng, device, m, 512))
            want = linear_int8(*quantize_int8_rows(x), w, sw)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("m", [3, 40, 300, 700])
def test_linear_scales_of_far_apart_sizes(nq, device, m):
    """Large activations against small weights: the result fits bf16 where sum * sx would not fit fp32."""

    from nari_qwen3_tts_amd.layers import linear_int8

    rng = np.random.default_rng(m)
    n = 3000 if m == 700 else 96
    q, w = _codes(rng, device, m, 512), _codes(rng, device, n, 512)
    s = torch.from_numpy(rng.uniform(1e35, 1e36, m).astype(np.float32)).to(device)
    sw = torch.from_numpy(rng.uniform(1e-6, 1e-5, n).astype(np.float32)).to(device)
    _check(linear_int8(q, s, w, sw), q, s, w, sw)


@pytest.mark.parametrize("m,n,k,tile", [
    (640, 12288, 2048, (128, 256)), (4001, 2040, 1040, (128, 256)), (2050, 2100, 384, (128, 256)),
    (2050, 2100, 400, (128, 256)), (2050, 2100, 512, (128, 256)), (2050, 2100, 528, (128, 256)),
    (2050, 2100, 16, (128, 256)), (1900, 2305, 6144, (128, 256)),
    (300, 5001, 2064, (64, 128)), (640, 6144, 1040, (64, 128)), (250, 4090, 1552, (64, 64)), (129, 700, 6160, (32, 16)),
    (64, 4096, 2064, (64, 16)), (50, 2040, 1040, (32, 16)), (16, 5000, 3088, (16, 16)),
])
def test_linear_long_sums(nq, device, m, n, k, tile):
    """Each kernel through its loop over whole stages, around the loop's bounds and with a part of a stage behind it."""

    from nari_qwen3_tts_amd import _lib
    from nari_qwen3_tts_amd.layers import linear_int8

    assert _lib.load().nq_linear_int8_tile(m, n) == tile[0] << 16 | tile[1]
    rng = np.random.default_rng(m + n + k)
    q, w = _codes(rng, device, m, k), _codes(rng, device, n, k)
    s, sw = torch.rand(m, device=device) + 0.01, torch.rand(n, device=device) + 0.01
    out = torch.full((m, n + 8), 7.0, dtype=torch.bfloat16, device=device)
    linear_int8(q, s, w, sw, out=out[:, :n])
    assert (out[:, n:] == 7.0).all()
    _check(out[:, :n], q, s, w, sw)
    again = linear_int8(q, s, w, sw)
    assert torch.equal(again.view(torch.int16), out[:, :n].contiguous().view(torch.int16))


def test_quantize_every_quotient(nq, device):
    """Every significand under every maximum's, eleven exponents down (below them every code is 0), both signs, against integer
    arithmetic; the same rows near the ends of bf16's range."""

    from nari_qwen3_tts_amd.layers import quantize_int8_rows

    a, k, b = np.arange(128, 256), np.arange(11), np.arange(128, 256)
    x = (a[None, :] * 2.0 ** -k[:, None].astype(np.float64)).reshape(-1)  # [11 * 128]
    rows = np.minimum(x, b[:, None])  # what lies above a row's maximum is the maximum
    rows[:, 1::2] *= -1
    rows = np.concatenate((rows, np.repeat(b[:, None], 16, 1)), 1)
    halves = np.abs(rows) * 2**10  # integers
    num, den = (254 * halves).astype(np.int64), (b[:, None] << 10).astype(np.int64)
    whole, rest = num // (2 * den), num % (2 * den)
    codes = np.sign(rows) * (whole + ((rest > den) | ((rest == den) & (whole % 2 == 1))))
    for power in (0, 100, 119, -60, -100):
        t = torch.from_numpy(rows * 2.0**power).to(device).to(torch.bfloat16)
        assert np.array_equal(to_np(t), (rows * 2.0**power).astype(np.float32))  # bf16 holds them
        q, s = quantize_int8_rows(t)
        assert np.array_equal(q.cpu().numpy(), codes)
        assert torch.equal(s.cpu(), torch.from_numpy((b * 2.0**power).astype(np.float32) / np.float32(127)))


@pytest.mark.parametrize("m,n,k", [(48, 4090, 2064), (77, 2041, 3088), (33, 2300, 1024), (140, 1300, 16)])
def test_linear_long_sums_in_pieces_of_48_rows(nq, device, m, n, k):
    test_linear_long_sums(nq, device, m, n, k, (48, 16))
