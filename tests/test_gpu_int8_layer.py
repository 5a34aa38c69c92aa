"""A layer behind its attention and a step's end, as they follow one another: the output projection with a bias, the
add-norm in int8 codes, the perceptron's products onto the residual, the last norm, the head and the draw.  Each
operator is checked against its oracle fed the device's own inputs, so the bounds are the operators' own; then the run on
another stream, and captured, with other inputs and the program's own work between the replays."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import epilogue as o_epi
from oracle import int8 as o_int8
from oracle import sampler as o_samp

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _bf16(rng, device, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(device, torch.bfloat16)


class _Layer:
    """Weights of width ``k`` and a perceptron of ``inner``, a head of ``vocab``; buffers for ``rows``."""

    def __init__(self, rng, device, rows, k, inner, vocab):
        from nari_qwen3_tts_amd.layers import quantize_int8_rows

        def codes(n, width):
            return quantize_int8_rows(_bf16(rng, device, n, width, std=width**-0.5))

        self.rng, self.device, self.rows, self.k = rng, device, rows, k
        self.wo, self.bo = _bf16(rng, device, k, k, std=k**-0.5), _bf16(rng, device, k, std=0.1)
        self.norms = [(1.0 + _bf16(rng, device, k, std=0.2)).contiguous() for _ in range(2)]
        self.first, self.second, self.head = codes(2 * inner, k), codes(k, inner), codes(vocab, k)
        self.lift = _bf16(rng, device, vocab, std=0.5)
        self.context = torch.empty(rows, k, dtype=torch.bfloat16, device=device)
        self.residual = torch.empty_like(self.context)
        self.uniforms = torch.empty(rows, device=device)
        self.params = (torch.from_numpy(rng.choice([0.0, 0.6, 1.0], rows).astype(np.float32)).to(device),
                       torch.from_numpy(rng.choice([0, 1, 20], rows).astype(np.int32)).to(device),
                       torch.from_numpy(rng.choice([0.9, 1.0], rows).astype(np.float32)).to(device),
                       torch.from_numpy(rng.choice([0.0, 0.05], rows).astype(np.float32)).to(device))

    def fill(self):
        self.context.copy_(_bf16(self.rng, self.device, self.rows, self.k))
        self.residual.copy_(_bf16(self.rng, self.device, self.rows, self.k, std=3.0))
        self.uniforms.copy_(torch.from_numpy((self.rng.integers(0, 1 << 24, self.rows) / (1 << 24)).astype(np.float32)))

    def run(self):
        """Every intermediate; the residual is updated in place, as a step does."""

        from nari_qwen3_tts_amd import layers
        from nari_qwen3_tts_amd.sampling import sample_min_p

        hidden = layers.linear_act(self.context, self.wo, self.bo)
        q, s = layers.add_rmsnorm_int8(hidden, self.residual, self.norms[0], EPS)
        middle = self.residual.clone()
        gate_up = layers.linear_int8(q, s, *self.first)
        inner = layers.silu_mul(gate_up)
        qi, si = layers.quantize_int8_rows(inner)
        layers.linear_int8(qi, si, *self.second, self.residual, residual=self.residual)
        qn, sn = layers.rmsnorm_int8(self.residual, self.norms[1], EPS)
        logits = layers.linear_int8(qn, sn, *self.head, bias=self.lift)
        tokens = sample_min_p(logits, *self.params, self.uniforms)
        return hidden, q, s, middle, gate_up, inner, qi, si, self.residual.clone(), qn, sn, logits, tokens


def _np(t):
    return to_np(t).astype(np.float64)


def _product(out, codes, weight, bias=None, residual=None):
    y = o_int8.linear(*(t.cpu().numpy() for t in (*codes, *weight)))
    bias, residual = (None if t is None else _np(t) for t in (bias, residual))
    bound = o_epi.bound(y, 4 * 2.0**-24 * np.abs(y), bias, None, residual)
    assert (np.abs(_np(out) - o_epi.product(y, bias, None, residual)) <= bound).all()


def _scales(got, want, width):
    # the bound of a norm's scales, width / 64 squares a lane and 10 additions of the lanes, the root, its product and quotient
    assert (np.abs(got.cpu().numpy() - want) <= ((width / 64 + 12) / 2 + 4) * 2.0**-24 * want).all()


def _check(layer, residual, got):
    hidden, q, s, middle, gate_up, inner, qi, si, after, qn, sn, logits, tokens = got
    x, w = _np(layer.context), _np(layer.wo)
    off = layer.k * 2.0**-24 * (np.abs(x) @ np.abs(w).T)
    bias = _np(layer.bo)
    assert (np.abs(_np(hidden) - o_epi.product(x @ w.T, bias)) <= o_epi.bound(x @ w.T, off, bias)).all()
    want = o_int8.add_rmsnorm(to_np(hidden), to_np(residual), to_np(layer.norms[0]), EPS)
    assert np.array_equal(to_np(middle), want[0]) and np.array_equal(q.cpu().numpy(), want[1])
    _scales(s, want[2], layer.k)
    _product(gate_up, (q, s), layer.first)
    want = o_int8.quantize_rows(to_np(inner))
    assert np.array_equal(qi.cpu().numpy(), want[0])
    _product(after, (qi, si), layer.second, None, middle)
    want = o_int8.add_rmsnorm(None, to_np(after), to_np(layer.norms[1]), EPS)
    assert np.array_equal(qn.cpu().numpy(), want[1])
    _scales(sn, want[2], layer.k)
    _product(logits, (qn, sn), layer.head, layer.lift)
    params = [p.cpu().tolist() for p in (*layer.params, layer.uniforms)]
    assert np.array_equal(tokens.cpu().numpy(), o_samp.sample_min_p(to_np(logits), *params))


@pytest.mark.parametrize("rows,k,inner,vocab", [(1, 2048, 6144, 2048), (9, 512, 1040, 5001), (77, 1024, 2048, 2051),
                                                (640, 2048, 1024, 4099)])
def test_a_layer_and_a_draw(nq, device, rows, k, inner, vocab):
    layer = _Layer(np.random.default_rng(rows + k), device, rows, k, inner, vocab)
    layer.fill()
    start = layer.residual.clone()
    want = layer.run()
    _check(layer, start, want)
    # another stream, the same bits
    layer.residual.copy_(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer.run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # the captured run, which updates the residual in place at each replay
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.run()
    for _ in range(3):
        layer.fill()
        start = layer.residual.clone()
        want = layer.run()
        layer.residual.copy_(start)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(layer.residual, want[8])


def test_rows_do_not_depend_on_the_batch(nq, device):
    """A row's codes and tokens alone are those it has in a batch: sums in 8 bits are exact at any number of rows."""

    from nari_qwen3_tts_amd import layers
    from nari_qwen3_tts_amd.sampling import sample_min_p

    layer = _Layer(np.random.default_rng(5), device, 130, 1024, 512, 3001)
    layer.fill()

    def run(part):
        residual = layer.residual[part].clone()
        q, s = layers.add_rmsnorm_int8(layer.context[part], residual, layer.norms[0], EPS)
        logits = layers.linear_int8(q, s, *layer.head, bias=layer.lift, activation="gelu")
        return q, s, logits, sample_min_p(logits, *(p[part] for p in layer.params), layer.uniforms[part])

    whole = run(slice(0, 130))
    for part in (slice(0, 1), slice(17, 18), slice(40, 77), slice(100, 130)):
        got = run(part)
        assert all(torch.equal(a, b[part]) for a, b in zip(got, whole))
