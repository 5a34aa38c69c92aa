"""Products with an epilogue against the float64 oracle.  Operands of small integers make the sums exact, so the bound
is the epilogue's alone; with ordinary values a sum of K bf16 products, each exact in fp32, is within K 2^-24 of
sum |x w| in any order."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import epilogue as o_epi
from oracle import int8 as o_int8

pytestmark = pytest.mark.gpu

ACTS = o_epi.ACTIVATIONS


def _bf16(rng, device, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(device, torch.bfloat16)


def _whole(rng, device, *shape):
    return torch.from_numpy(rng.integers(-4, 5, shape).astype(np.float32)).to(device, torch.bfloat16)


def _np(t):
    return None if t is None else to_np(t).astype(np.float64)


def _compare(out, y, off, bias, act, res):
    bias, res = _np(bias), _np(res)
    want, got = o_epi.product(y, bias, act, res), _np(out)
    bound = o_epi.bound(y, off, bias, act, res)
    assert (np.abs(got - want) <= bound).all(), (act, np.abs(got - want).max(), (np.abs(got - want) / bound).max())


def _check(out, x, w, bias=None, act=None, res=None, exact=True):
    x, w = _np(x), _np(w)
    off = 0.0 if exact else x.shape[1] * 2.0**-24 * (np.abs(x) @ np.abs(w).T)
    _compare(out, x @ w.T, off, bias, act, res)


def _check8(out, q, s, w, sw, bias=None, act=None, res=None):
    y = o_int8.linear(*(t.cpu().numpy() for t in (q, s, w, sw)))
    _compare(out, y, 4 * 2.0**-24 * np.abs(y), bias, act, res)


def _codes(rng, device, rows, k):
    return torch.from_numpy(rng.integers(-127, 128, (rows, k)).astype(np.int8)).to(device)


def _scales(rng, device, n, k):
    return torch.from_numpy((rng.uniform(0.3, 1.0, n) / np.sqrt(k) / 8).astype(np.float32)).to(device)


@pytest.mark.parametrize("n,k", [(16, 8), (1, 2048), (50, 136), (257, 1032), (1024, 2048), (130, 6144), (2048, 64)])
@pytest.mark.parametrize("m", [1, 2, 16, 17, 33, 64, 65, 100, 129, 300])
def test_bf16(nq, device, m, n, k):
    from nari_qwen3_tts_amd.layers import linear_act

    rng = np.random.default_rng(m * 7 + n + k)
    x, w = _whole(rng, device, m, k), _whole(rng, device, n, k) * 2.0**-7
    bias, res = _bf16(rng, device, n), _bf16(rng, device, m, n, std=3.0)
    for i, act in enumerate(ACTS):
        b, r = (bias, None, bias, None)[(i + m) % 4], (res, res, None, None)[(i + m) % 4]
        out = linear_act(x, w, bias=b, activation=act, residual=r)
        _check(out, x, w, b, act, r)
    x, w = _bf16(rng, device, m, k), _bf16(rng, device, n, k, std=k**-0.5)
    _check(linear_act(x, w, bias, "gelu", res), x, w, bias, "gelu", res, exact=False)


@pytest.mark.parametrize("n,k", [(16, 16), (1, 2048), (50, 144), (257, 1040), (1024, 2048), (130, 6144), (2048, 128)])
@pytest.mark.parametrize("m", [1, 2, 16, 17, 33, 64, 65, 100, 129, 300])
def test_int8(nq, device, m, n, k):
    from nari_qwen3_tts_amd.layers import linear_int8

    rng = np.random.default_rng(m * 7 + n + k)
    q, w = _codes(rng, device, m, k), _codes(rng, device, n, k)
    s, sw = _scales(rng, device, m, k), torch.rand(n, device=device) * 0.02 + 0.001
    bias, res = _bf16(rng, device, n), _bf16(rng, device, m, n, std=3.0)
    for i, act in enumerate(ACTS):
        b, r = (bias, None, bias, None)[(i + m) % 4], (res, res, None, None)[(i + m) % 4]
        out = linear_int8(q, s, w, sw, bias=b, activation=act, residual=r)
        _check8(out, q, s, w, sw, b, act, r)
        assert torch.equal(out[-1], linear_int8(q[-1:], s[-1:], w, sw, bias=b, activation=act,
                                                residual=None if r is None else r[-1:])[0])


@pytest.mark.parametrize("m,n,k", [
    (640, 12288, 2048), (4001, 2040, 520), (2050, 2100, 192), (2050, 2100, 200), (2050, 2100, 256), (2050, 2100, 264),
    (2050, 2100, 8), (1900, 2305, 3080), (300, 5001, 1032), (640, 6144, 520), (250, 4090, 776), (129, 700, 3088),
    (64, 4096, 1032), (50, 2040, 520), (16, 5000, 1544), (4001, 6144, 2048), (1430, 2001, 8), (1430, 2001, 200),
    (1430, 2001, 264), (500, 6100, 1544), (48, 4090, 1032), (77, 2041, 1544),
])
def test_large(nq, device, m, n, k):
    """Each kernel through its loop over whole stages, around the loop's bounds and with a part of a stage behind it."""

    from nari_qwen3_tts_amd.layers import linear_act, linear_int8

    rng = np.random.default_rng(m + n + k)
    x, w = _whole(rng, device, m, k), _whole(rng, device, n, k) * 2.0**-7
    bias, res = _bf16(rng, device, n), _bf16(rng, device, m, n)
    out = torch.full((m, n + 8), 7.0, dtype=torch.bfloat16, device=device)
    linear_act(x, w, bias, "silu", res, out=out[:, :n])
    assert (out[:, n:] == 7.0).all()
    _check(out[:, :n], x, w, bias, "silu", res)
    again = linear_act(x, w, bias, "silu", res)
    assert torch.equal(again.view(torch.int16), out[:, :n].contiguous().view(torch.int16))
    q, wq = _codes(rng, device, m, 2 * k), _codes(rng, device, n, 2 * k)
    s, sw = _scales(rng, device, m, 2 * k), torch.rand(n, device=device) * 0.02 + 0.001
    _check8(linear_int8(q, s, wq, sw, bias=bias, residual=res), q, s, wq, sw, bias, None, res)


@pytest.mark.parametrize("m", [1, 3, 40, 200, 700])
@pytest.mark.parametrize("n", [77, 1280])
def test_strided(nq, device, m, n):
    """Slices of wider rows, residuals and outputs at odd addresses, one residual row for all; neighbours stay."""

    from nari_qwen3_tts_amd.layers import linear_act, linear_int8

    rng = np.random.default_rng(m + n)
    x, w = _whole(rng, device, m, 288)[:, 16:256], _whole(rng, device, n, 272)[:, 32:]
    q, wq = _codes(rng, device, m, 288)[:, 16:256], _codes(rng, device, n, 272)[:, 32:]
    s, sw = _scales(rng, device, m, 240), torch.rand(n, device=device)
    wide = _bf16(rng, device, m, n + 9)
    bias = _bf16(rng, device, n + 1)[1:]
    for at in (0, 3, 8):
        out = torch.full((m, n + 16), 7.0, dtype=torch.bfloat16, device=device)
        for res in (wide[:, at:at + n], wide[:1, 1:n + 1].expand(m, n), None):
            part = out[:, at:at + n]
            linear_act(x, w, bias, "relu", res, out=part)
            _check(part, x, w, bias, "relu", res)
            linear_int8(q, s, wq, sw, part, bias=bias, residual=res)
            _check8(part, q, s, wq, sw, bias, None, res)
            assert (out[:, :at] == 7.0).all() and (out[:, at + n:] == 7.0).all()


@pytest.mark.parametrize("m", [1, 20, 100, 900])
def test_onto_the_residual_itself(nq, device, m):
    from nari_qwen3_tts_amd.layers import linear_act, linear_int8

    rng = np.random.default_rng(m)
    x, w = _whole(rng, device, m, 512), _whole(rng, device, 1000, 512) * 2.0**-7
    q, wq = _codes(rng, device, m, 512), _codes(rng, device, 1000, 512)
    s, sw = _scales(rng, device, m, 512), torch.rand(1000, device=device)
    for width in (1000, 1003):
        stream = _bf16(rng, device, m, width)[:, :1000]
        before = stream.clone()
        assert linear_act(x, w, activation="gelu_tanh", residual=stream, out=stream).data_ptr() == stream.data_ptr()
        _check(stream, x, w, None, "gelu_tanh", before)
        before = stream.clone()
        linear_int8(q, s, wq, sw, stream, residual=stream)
        _check8(stream, q, s, wq, sw, None, None, before)


@pytest.mark.parametrize("act", ACTS)
def test_every_value(nq, device, act):
    """Each finite bf16 value through each activation."""

    from nari_qwen3_tts_amd.layers import linear_act

    values = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    values = values[values.isfinite()]
    x = torch.zeros(len(values), 8, dtype=torch.bfloat16, device=device)
    x[:, 3] = values.to(device)
    w = torch.zeros(1, 8, dtype=torch.bfloat16, device=device)
    w[0, 3] = 1
    out = linear_act(x, w, activation=act)
    # the matrix unit takes subnormal operands as zeros or as they are: below the bound's last term either way
    _check(out, x, w, None, act)


@pytest.mark.parametrize("m", [20, 150, 900])
def test_odd_values_stay_in_their_rows_and_columns(nq, device, m):
    from nari_qwen3_tts_amd.layers import linear_act, linear_int8

    rng = np.random.default_rng(m)
    x, w, n = _bf16(rng, device, m, 72), _bf16(rng, device, 300, 72, std=0.1), 300
    bias, res = _bf16(rng, device, n), _bf16(rng, device, m, n)
    x[m - 1, 5], x[3, 71], w[n - 1, 0], bias[7], res[2, 9] = (float("nan"),) * 5
    for act in ACTS:
        out = linear_act(x, w, bias, act, res)
        bad = torch.zeros(m, n, dtype=torch.bool, device=device)
        bad[m - 1] = bad[3] = bad[2, 9] = True
        bad[:, n - 1] = bad[:, 7] = True
        assert torch.equal(out.isnan(), bad), act
    q, wq = _codes(rng, device, m, 80), _codes(rng, device, n, 80)
    s, sw = _scales(rng, device, m, 80), torch.rand(n, device=device)
    s[4], sw[11] = float("nan"), float("nan")
    out = linear_int8(q, s, wq, sw, activation="silu", residual=res)
    bad = torch.zeros(m, n, dtype=torch.bool, device=device)
    bad[4] = bad[2, 9] = True
    bad[:, 11] = True
    assert torch.equal(out.isnan(), bad)


def test_offsets_past_32_bits(nq, device):
    from nari_qwen3_tts_amd.layers import linear_act

    rng = np.random.default_rng(6)
    big = torch.zeros(70, 1 << 26, dtype=torch.bfloat16, device=device)
    x, w, res = big[:, :128], big[:, 1 << 20:][:, :128], big[:, 1 << 21:][:, :70]
    x.copy_(_whole(rng, device, 70, 128))
    w.copy_(_whole(rng, device, 70, 128))
    res.copy_(_bf16(rng, device, 70, 70))
    out = torch.zeros(70, 1 << 26, dtype=torch.bfloat16, device=device)[:, :70]
    for rows in (70, 64):
        linear_act(x[:rows], w, residual=res[:rows], out=out[:rows])
        _check(out[:rows], x[:rows], w, None, None, res[:rows])


def test_streams_graphs_and_no_rows(nq, device):
    from nari_qwen3_tts_amd.layers import linear_act, linear_int8

    rng = np.random.default_rng(7)
    for m in (8, 300, 1500):
        n, k = 1030, 512
        x, w = _bf16(rng, device, m, k), _bf16(rng, device, n, k)
        q, wq = _codes(rng, device, m, k), _codes(rng, device, n, k)
        s, sw = _scales(rng, device, m, k), torch.rand(n, device=device)
        bias, res = _bf16(rng, device, n), _bf16(rng, device, m, n)
        out, out8 = torch.empty_like(res), torch.empty_like(res)

        def both(a=None, b=None):
            return (linear_act(x, w, bias, "silu", res, out=a),
                    linear_int8(q, s, wq, sw, b, bias=bias, activation="gelu", residual=res))

        want = both()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both(out, out8)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, want[0]) and torch.equal(out8, want[1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            both(out, out8)
        for _ in range(3):
            x.copy_(_bf16(rng, device, m, k))
            q.copy_(_codes(rng, device, m, k))
            res.copy_(_bf16(rng, device, m, n))
            want = both()
            out.zero_()
            out8.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(out8, want[1])
    assert linear_act(x[:0], w, bias, "silu", res[:0]).shape == (0, n)
    assert linear_act(x, w[:0], residual=res[:, :0]).shape == (1500, 0)
    assert linear_int8(q[:0], s[:0], wq, sw, bias=bias).shape == (0, n)
