"""The epilogue's oracle against torch's functions, and the entry points' refusals (no GPU needed)."""

from __future__ import annotations

import re

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import epilogue as o_epi


def test_activations_against_torch():
    y = torch.linspace(-12, 12, 4001, dtype=torch.float64)
    for name, fn in ((None, lambda t: t), ("relu", F.relu), ("gelu", F.gelu), ("silu", F.silu),
                     ("gelu_tanh", lambda t: F.gelu(t, approximate="tanh"))):
        want = fn(y).numpy()
        assert np.abs(o_epi.activate(y.numpy(), name) - want).max() <= 1e-14 * 12
    assert o_epi.activate(np.array([-40.0]), "silu")[0] == pytest.approx(-40 * np.exp(-40), rel=1e-12)
    # slopes, on which the bound relies, by differences
    for name in o_epi.ACTIVATIONS:
        assert np.abs(np.diff(o_epi.activate(y.numpy(), name)) / np.diff(y.numpy())).max() < 1.2


def test_product_order():
    y = o_epi.product(np.array([[1.0, -3.0]]), [1.0, 1.0], "relu", [[-5.0, 7.0]])
    assert y.tolist() == [[-3.0, 7.0]]


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


_EPILOGUE = [
    (dict(activation="tanh"), ValueError),
    (dict(activation=1), ValueError),
    (dict(bias=torch.zeros(3)), TypeError),
    (dict(bias=_bf(4)), ValueError),
    (dict(bias=_bf(6)[::2]), ValueError),
    (dict(residual=torch.zeros(2, 3)), TypeError),
    (dict(residual=_bf(2, 4)), ValueError),
    (dict(residual=_bf(3, 2).t()), ValueError),
    (dict(out=torch.zeros(2, 3)), ValueError),
    (dict(out=_bf(2, 4)), ValueError),
    (dict(out=_bf(3, 2).t()), ValueError),
    (dict(), ValueError),  # the call itself, but on the CPU
]


@pytest.mark.parametrize("change,error", _EPILOGUE + [
    (dict(x=torch.zeros(2, 32)), TypeError),
    (dict(weight=torch.zeros(3, 32)), TypeError),
    (dict(x=_bf(32)), ValueError),
    (dict(x=_bf(32, 2).t()), ValueError),
    (dict(weight=_bf(32, 3).t()), ValueError),
    (dict(weight=_bf(3, 40)), ValueError),
    (dict(x=_bf(2, 12), weight=_bf(3, 12)), ValueError),
    (dict(x=_bf(2, 0), weight=_bf(3, 0)), ValueError),
])
def test_linear_act_refusals(nq, change, error):
    from nari_qwen3_tts_amd.layers import linear_act

    with pytest.raises(error):
        linear_act(**{**dict(x=_bf(2, 32), weight=_bf(3, 32)), **change})


@pytest.mark.parametrize("change,error", _EPILOGUE)
def test_linear_int8_epilogue_refusals(nq, change, error):
    from nari_qwen3_tts_amd.layers import linear_int8

    args = dict(q=torch.zeros(2, 32, dtype=torch.int8), scales=torch.zeros(2),
                weight_q=torch.zeros(3, 32, dtype=torch.int8), weight_scales=torch.zeros(3))
    with pytest.raises(error):
        linear_int8(**{**args, **change})


def test_activation_codes_agree_with_the_header(nq):
    from test_abi import HEADER

    from nari_qwen3_tts_amd import _lib, layers

    body = re.search(r"enum nq_activation \{([^}]*)\}", HEADER.read_text()).group(1)
    declared = {k.strip(): int(v) for k, v in (e.split("=") for e in body.split(","))}
    assert declared == {k: getattr(_lib, k) for k in declared}
    assert list(layers.ACTIVATIONS.values()) == sorted(declared.values()) and tuple(layers.ACTIVATIONS) == o_epi.ACTIVATIONS


def test_host_checks_of_the_product_entries(nq):
    """Refused before any launch (placeholder pointers)."""

    from nari_qwen3_tts_amd import _lib

    lib = _lib.load()

    def bf16(x=16, x_s0=64, w=16, w_s0=64, m=2, n=3, k=64, bias=None, act=0, res=None, r_s0=3, out=16, o_s0=3):
        return lib.nq_linear_act(x, x_s0, w, w_s0, m, n, k, bias, act, res, r_s0, out, o_s0, None)

    def int8(x=16, x_s0=64, w=16, w_s0=64, m=2, n=3, k=64, bias=None, act=0, res=None, r_s0=3, out=16, o_s0=3, s=16):
        return lib.nq_linear_int8_act(x, x_s0, s, w, w_s0, s, m, n, k, bias, act, res, r_s0, out, o_s0, None)

    for call in (bf16, int8):
        assert call(m=0) == 0 and call(n=0) == 0
        for bad in (dict(m=-1), dict(x=None), dict(w=None), dict(out=None), dict(k=0), dict(o_s0=2), dict(act=5),
                    dict(act=-1), dict(res=16, r_s0=-1), dict(x_s0=-64), dict(w_s0=-64)):
            assert call(**bad) == -1, bad
        for bad in (dict(k=68), dict(x=8), dict(w=8), dict(x_s0=68), dict(w_s0=68), dict(out=3), dict(bias=3),
                    dict(res=3), dict(m=0x7fffffff, n=0x7fffffff, o_s0=1 << 32)):
            assert call(**bad) == -2, bad
    assert bf16(k=(1 << 24) + 8, x_s0=1 << 25, w_s0=1 << 25) == -2 and bf16(k=4) == -1
    assert int8(k=(1 << 17) + 16, x_s0=1 << 18, w_s0=1 << 18) == -2 and int8(k=8) == -1 and int8(s=None) == -1
    assert int8(s=2) == -2
