"""Oracle for products with a bias, an activation and a residual in their epilogue (test infrastructure only), float64.

``bound`` is how far a kernel may be that computes the epilogue in fp32 from a sum ``off`` away from the exact one.
Pinned by tests/test_oracle_epilogue.py against torch's own functions and closed forms.
"""

from __future__ import annotations

import numpy as np
from scipy.special import erfc, expit

ACTIVATIONS = (None, "relu", "gelu", "gelu_tanh", "silu")
_TANH = 2.0 * np.sqrt(2.0 / np.pi)


def activate(y: np.ndarray, activation: str | None) -> np.ndarray:
    y = np.asarray(y, np.float64)
    if activation == "relu":
        return np.where(y < 0, 0.0, y)
    if activation == "gelu":
        return 0.5 * y * erfc(-y * np.sqrt(0.5))
    if activation == "gelu_tanh":
        return y * expit(_TANH * (y + 0.044715 * y**3))
    return y * expit(y) if activation == "silu" else y


def product(y: np.ndarray, bias=None, activation=None, residual=None) -> np.ndarray:
    y = y if bias is None else y + np.asarray(bias, np.float64)
    y = activate(y, activation)
    return y if residual is None else y + np.asarray(residual, np.float64)


def bound(y: np.ndarray, off, bias=None, activation=None, residual=None) -> np.ndarray:
    """|kernel - product(y, ...)| in bf16 units and below: the half step of the result (2^-8 of it), what is off before
    the activation (``off`` and the bias's rounding) times its slope (below 1.2), the activation's own error and the
    residual's rounding.  An activation is a product with a factor f: with its argument z off by 2^-22 of itself, f is
    off by at most that times |z| (the logistic function) or 2 z^2 (erfc), and by 16 roundings of 2^-24 besides."""

    z = np.asarray(y, np.float64) if bias is None else y + np.asarray(bias, np.float64)
    v = activate(z, activation)
    before = 1.2 * (np.asarray(off) + 2.0**-23 * np.abs(z))
    if activation in ("silu", "gelu_tanh", "gelu"):
        with np.errstate(over="ignore"):
            arg = {"silu": np.abs(z), "gelu_tanh": np.abs(_TANH * (z + 0.044715 * z**3)), "gelu": z * z}[activation]
        # past this the factor is 1, or so small that it and its error are below the last term
        before = before + np.abs(v) * (np.minimum(arg, 120.0) + 4.0) * 2.0**-22
    want = v if residual is None else v + np.asarray(residual, np.float64)
    return 2.0**-8 * (np.abs(want) + before) + before + 2.0**-23 * np.abs(v) + 1e-30
