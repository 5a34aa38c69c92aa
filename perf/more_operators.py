"""Performance cases of the operators between a layer's attention blocks and at a step's end: the RMS norm with the
residual's addition that answers int8 codes and a scale a token, the matrix product with bias, activation and residual
in its epilogue (bf16 operands, or int8 codes with their scales), and the draw of a token with temperature, min-p,
top-k and top-p from a given random number, over vocabularies of any size.

Each case is one call as a serving step makes it.  Where ``own`` is false ``run`` restates the operator in
elementary torch operations; ``exact`` restates it in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # one listener's stream: a layer's norm, where launches and latency count
        {"name": "norm-1", "kind": "norm", "rows": 1, "width": 2048},
        # the headline batch, at the code predictor's width
        {"name": "norm-64", "kind": "norm", "rows": 64, "width": 1024},
        # a long prompt's chunk
        {"name": "norm-4001", "kind": "norm", "rows": 4001, "width": 2048},
        # one stream through a projection with a bias, as the code predictor's input takes it
        {"name": "bf16-1", "kind": "linear", "type": "bf16", "rows": 1, "out": 1024, "in": 2048, "bias": True,
         "act": "silu", "residual": False},
        # a batch of odd size through a down projection onto its residual
        {"name": "bf16-77", "kind": "linear", "type": "bf16", "rows": 77, "out": 2048, "in": 6144, "bias": False,
         "act": "none", "residual": True},
        # a long prompt's chunk through a perceptron's first half
        {"name": "bf16-4001", "kind": "linear", "type": "bf16", "rows": 4001, "out": 6144, "in": 2048, "bias": True,
         "act": "gelu_tanh", "residual": False},
        # one stream's down projection, the activations already in codes
        {"name": "int8-1", "kind": "linear", "type": "int8", "rows": 1, "out": 2048, "in": 6144, "bias": False,
         "act": "none", "residual": True},
        # the largest prefill bucket through a perceptron's first half
        {"name": "int8-640", "kind": "linear", "type": "int8", "rows": 640, "out": 6144, "in": 2048, "bias": True,
         "act": "silu", "residual": False},
        # a long prompt's chunk onto its residual
        {"name": "int8-4001", "kind": "linear", "type": "int8", "rows": 4001, "out": 2048, "in": 6144, "bias": True,
         "act": "none", "residual": True},
        # one stream's draw from the codec head
        {"name": "sample-1", "kind": "sample", "rows": 1, "vocab": 2048, "type": "bf16"},
        # the headline batch over the text vocabulary's order of size
        {"name": "sample-64", "kind": "sample", "rows": 64, "vocab": 65537, "type": "bf16"},
        # a large batch over a large vocabulary, logits in 32 bits
        {"name": "sample-256", "kind": "sample", "rows": 256, "vocab": 131072, "type": "fp32"},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    kind = rng.choice(("norm", "linear", "linear", "sample"))
    if kind == "norm":
        width = 16 * _log(rng, 4, 512)
        return {"kind": kind, "rows": _log(rng, 1, min(6000, 8_000_000 // width)), "width": width}
    if kind == "sample":
        vocab = _log(rng, 2, 200_000)
        return {"kind": kind, "rows": _log(rng, 1, min(256, 30_000_000 // vocab)), "vocab": vocab,
                "type": rng.choice(("bf16", "fp32"))}
    out, inner = _log(rng, 16, 6200), 16 * _log(rng, 4, 400)
    return {"kind": kind, "type": rng.choice(("bf16", "int8")),
            "rows": _log(rng, 1, min(4000, 48_000_000_000 // (out * inner))), "out": out, "in": inner,
            "bias": rng.random() < 0.6, "act": rng.choice(ACTIVATIONS), "residual": rng.random() < 0.5}


# -- inputs ------------------------------------------------------------------------------------------


def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + salt) % (1 << 62))
    return g


def _normal(g, *shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)


def _norm_inputs(case, seed):
    g, shape = _generator(seed, 1), (case["rows"], case["width"])
    # the residual stream is wider than what a block adds to it, and some of its channels are wider than the others
    spread = torch.exp2(_normal(g, case["width"]))
    return {"hidden": _normal(g, *shape).to(torch.bfloat16), "residual": (_normal(g, *shape) * spread * 4).to(torch.bfloat16),
            "norm_weight": (1.0 + _normal(g, case["width"], std=0.2)).to(torch.bfloat16)}


def _codes(x):
    """Codes rint(127 x / max |x|) and scales max |x| / 127 of each row."""

    top = x.abs().amax(-1, keepdim=True)
    return (x * 127.0 / top).round().to(torch.int8), (top / 127.0).squeeze(-1)


def _linear_inputs(case, seed):
    g, m, n, k = _generator(seed, 2), case["rows"], case["out"], case["in"]
    x = _normal(g, m, k) * torch.exp2(_normal(g, k, std=0.5))  # channels differ, as behind a norm's weight
    w = _normal(g, n, k, std=0.02)
    s = {"act": case["act"], "bias": _normal(g, n, std=0.5).to(torch.bfloat16) if case["bias"] else None,
         "onto": _normal(g, m, n, std=3.0).to(torch.bfloat16) if case["residual"] else None}
    if case["type"] == "bf16":
        return {**s, "x": x.to(torch.bfloat16), "weight": w.to(torch.bfloat16)}
    (q, scales), (wq, weight_scales) = _codes(x), _codes(w)
    return {**s, "q": q, "scales": scales, "weight_q": wq, "weight_scales": weight_scales}


def _sample_inputs(case, seed):
    g, rows, vocab = _generator(seed, 3), case["rows"], case["vocab"]
    # a bulk of unlikely tokens and some that stand out, rows more and less decided
    logits = _normal(g, rows, vocab) * torch.empty(rows, 1, device="cuda").uniform_(1.0, 3.0, generator=g)
    high = torch.empty(rows, vocab, device="cuda").uniform_(generator=g) < min(0.25, 40.0 / vocab)
    logits = logits + high * torch.empty(rows, vocab, device="cuda").uniform_(2.0, 8.0, generator=g)
    logits = logits.to(torch.bfloat16 if case["type"] == "bf16" else torch.float32)

    def some(values, dtype):
        at = torch.randint(len(values), (rows,), device="cuda", generator=g)
        return torch.tensor(values, dtype=dtype, device="cuda")[at]

    return {"logits": logits, "temperature": some((0.0, 0.6, 0.8, 0.9, 1.0, 1.0, 1.3), torch.float32),
            "top_k": some((0, 0, 0, 20, 50, 400), torch.int32), "top_p": some((1.0, 1.0, 0.95, 0.8), torch.float32),
            "min_p": some((0.0, 0.02, 0.05, 0.1, 0.3), torch.float32),
            "uniforms": torch.empty(rows, device="cuda").uniform_(generator=g)}


def prepare(case, seed):
    return {"norm": _norm_inputs, "linear": _linear_inputs, "sample": _sample_inputs}[case["kind"]](case, seed)


# -- one pass ----------------------------------------------------------------------------------------


def _norm(s):
    """Plain form.  The codes in 64 bits: the quotients lie next to ties."""

    x = (s["residual"].float() + s["hidden"].float()).to(torch.bfloat16)
    s["residual"].copy_(x)
    weighted = x.double() * s["norm_weight"].double()
    top = weighted.abs().amax(-1, keepdim=True)
    codes = (weighted * 127.0 / top).round().float()
    x = x.float()
    scales = top.float() * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) / 127.0
    return codes * scales, s["residual"]


def _activate(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y / (1.0 + torch.exp(-y)) if act == "silu" else y


def _linear(s):
    if "x" in s:
        y = s["x"].float() @ s["weight"].float().t()
    else:
        y = (s["q"].float() @ s["weight_q"].float().t()) * s["scales"][:, None] * s["weight_scales"]
    y = _activate(y if s["bias"] is None else y + s["bias"].float(), s["act"])
    return (y if s["onto"] is None else y + s["onto"].float()).to(torch.bfloat16)


def _sample(s):
    """Plain form in 64 bits, since the draw compares sums: the tokens in order of their logits (ties: the lowest id
    first), the prefix that min-p and top-k leave, of that the least whose mass reaches top_p of it, and the first token
    by id at which the kept mass reaches the uniform's share."""

    x = s["logits"].double()
    vocab, greedy = x.shape[1], s["temperature"] == 0
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    e = torch.exp((x - x[:, :1]) / t)
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    rank = torch.arange(vocab, device=x.device)
    e = torch.where((rank < k) & (e >= s["min_p"].double()[:, None]), e, 0.0)
    cum = e.cumsum(1)
    e = torch.where((rank == 0) | (cum - e < s["top_p"].double()[:, None] * cum[:, -1:]), e, 0.0)
    e = torch.zeros_like(e).scatter_(1, order, e)
    cum = e.cumsum(1)
    reached = (e > 0) & (cum >= s["uniforms"].double()[:, None] * cum[:, -1:])
    return torch.where(greedy, order[:, 0], torch.where(reached, rank, vocab).amin(1))


def _package():
    from __graft_entry__ import load_package

    load_package()
    from nari_qwen3_tts_amd import layers, sampling

    return layers, sampling


def _run_own(s):
    layers, sampling = _package()
    if "hidden" in s:
        q, scales = layers.add_rmsnorm_int8(s["hidden"], s["residual"], s["norm_weight"], EPS)
        return q * scales[:, None], s["residual"]
    if "logits" in s:
        return sampling.sample_min_p(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniforms"])
    act = None if s["act"] == "none" else s["act"]
    if "x" in s:
        return layers.linear_act(s["x"], s["weight"], bias=s["bias"], activation=act, residual=s["onto"])
    return layers.linear_int8(s["q"], s["scales"], s["weight_q"], s["weight_scales"], bias=s["bias"], activation=act,
                              residual=s["onto"])


def run(s):
    if own:
        return _run_own(s)
    return _norm(s) if "hidden" in s else _sample(s) if "logits" in s else _linear(s)


def work(case):
    rows = case["rows"]
    if case["kind"] == "norm":
        # both inputs in, the new residual, the codes and the scale out
        return {"bytes": rows * (7 * case["width"] + 4) + 2 * case["width"], "flops": 8 * rows * case["width"]}
    if case["kind"] == "sample":
        return {"bytes": rows * (case["vocab"] * (2 if case["type"] == "bf16" else 4) + 28), "flops": 4 * rows * case["vocab"]}
    n, k, int8 = case["out"], case["in"], case["type"] == "int8"
    return {"bytes": (rows + n) * (k + 4 if int8 else 2 * k) + 2 * rows * n * (1 + case["residual"]) + 2 * n * case["bias"],
            "flops": 2 * rows * n * k}


# -- the same in 64 bits -------------------------------------------------------------------------------


def _exact_norm(case, seed):
    s = _norm_inputs(case, seed)
    x = (s["residual"].double() + s["hidden"].double()).to(torch.bfloat16).double()  # bf16's sums are exact in 64 bits
    y = x / torch.sqrt(torch.mean(torch.square(x), -1, keepdim=True) + EPS) * s["norm_weight"].double()
    # the codes from x times weight, whose quotients the norm's own rounding does not move off a tie
    p = x * s["norm_weight"].double()
    codes = torch.round(127.0 * p / torch.linalg.vector_norm(p, ord=math.inf, dim=-1, keepdim=True))
    return codes * (torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True) / 127.0), x


def _exact_linear(case, seed):
    s = _linear_inputs(case, seed)
    if case["type"] == "bf16":
        x, w = s["x"].double(), s["weight"].double()
    else:
        x, w = s["q"].double() * s["scales"].double()[:, None], s["weight_q"].double() * s["weight_scales"].double()[:, None]
    y = torch.matmul(x, w.t())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == "relu":
        y = torch.maximum(y, torch.zeros_like(y))
    elif case["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    elif case["act"] == "gelu_tanh":
        y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y**3))  # (1 + tanh z) / 2
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    return y if s["onto"] is None else y + s["onto"].double()


def exact(case, seed):
    if case["kind"] == "sample":
        return None  # tokens: whole numbers
    return (_exact_norm if case["kind"] == "norm" else _exact_linear)(case, seed)
