"""The operators around the products of a decoder layer served from 4-bit weights: a product with its
epilogue (bias, activation, gate, residual), the norm with the residual's addition, and a
mixture-of-experts layer (its router, its experts).

Each case is measured in one of two forms: the framework's own calls (`own` true), or the same
mathematics in elementary torch operations in 32 bits (`own` false).

A weight [N, K] is packed as int32 words: word ((n / 16) * (K / 64) + k / 64) * 128 + lane * 4 + s holds,
in nibble 4h + 2b + a, the code of row 16 (n / 16) + lane / 4 + 8a and column 64 (k / 64) + 16s +
2 (lane % 4) + 8b + h.  Scales are fp16 [K / G, N]; a weight is (code - 8) * scale.  A product's epilogue works
on fp16 weights (that value rounded once, as `w4a16_dequant` gives it); the experts' weights are the value
itself.  Rows of a gated weight alternate in runs of eight: eight of the gate, eight of the other factor.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _framework():
    path = os.path.join(_ROOT, "w4a16-gemm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import w4a16_opt
    return w4a16_opt


# ------------------------------------------------------------------------------ cases

def _linear(name, m, n, k, group, activation="none", gated=False, bias=False, residual=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "group": group, "activation": activation,
            "gated": gated, "bias": bias, "residual": residual}


def _norm(name, tokens, heads, dim, dtype, residual="none"):
    """heads 0: rows [tokens, dim]; otherwise the heads of a fused projection, [tokens, heads, dim]."""
    return {"name": name, "op": "norm", "tokens": tokens, "heads": heads, "dim": dim, "dtype": dtype,
            "residual": residual}


def _route(name, tokens, experts, k, dtype, renormalize=True, masked=False):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype,
            "renormalize": renormalize, "masked": masked}


def _experts(name, tokens, experts, k, hidden, inner, group, activation="silu", residual=False, skew=0.5):
    return {"name": name, "op": "experts", "tokens": tokens, "experts": experts, "k": k, "hidden": hidden,
            "inner": inner, "group": group, "activation": activation, "residual": residual, "skew": skew}


def listed():
    return [
        # the last product of a decoder layer for one token, Llama-3-8B: added to the residual stream
        _linear("linear down 1", 1, 4096, 14336, 128, residual=True),
        # gate and up in one product for eight sequences, Llama-3-8B
        _linear("linear gate up 8", 8, 28672, 4096, 128, "silu", gated=True),
        # a product with a bias, odd numbers of tokens and columns, fine groups
        _linear("linear bias gelu 77", 77, 4112, 4160, 64, "gelu", bias=True),
        # gate and up of a whole prompt
        _linear("linear gate up 2048", 2048, 28672, 4096, 128, "silu", gated=True),
        # the norm before a projection in a decode step of eight sequences: latency
        _norm("norm step 8", 8, 0, 4096, "fp16", "same"),
        # the norm of a long prompt, Llama-3-70B width: bandwidth
        _norm("norm prompt 8192", 8192, 0, 8192, "bf16", "same"),
        # the router of a decode step
        _route("route step 16", 16, 128, 8, "fp32"),
        # the router of a long prompt, an odd number of experts, some of them masked out
        _route("route prompt 8192", 8192, 60, 4, "bf16", renormalize=False, masked=True),
        # one token through large experts: bound by the two experts' weights
        _experts("experts 1 of 8 large", 1, 8, 2, 4096, 14336, 128),
        # one token through small experts: latency
        _experts("experts 1 of 128 small", 1, 128, 8, 2048, 768, 128, residual=True),
        # a decode step of 32 sequences, most experts touched by a token or two
        _experts("experts 32 of 64", 32, 64, 6, 2048, 1408, 128),
        # a prompt, loads of the experts uneven
        _experts("experts prompt 2048", 2048, 64, 6, 2048, 1408, 64, skew=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "route", "experts", "experts"])
    group = rng.choice([64, 128])
    if op == "linear":
        m = rng.choice([_log(rng, 1, 16), _log(rng, 1, 2048)])
        n = 16 * _log(rng, 1, 28672 // 16)
        k = group * _log(rng, 1, 14336 // group)
        while n * k > 28672 * 4096:
            n = 16 * max(1, n // 32)
        c = _linear("", m, n, k, group, rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), rng.random() < 0.4,
                    rng.random() < 0.5, rng.random() < 0.5)
    elif op == "norm":
        if rng.random() < 0.3:
            c = _norm("", _log(rng, 1, 4096), rng.choice([1, 2, 5, 8, 32, 40]), rng.choice([64, 128, 192, 256]),
                      rng.choice(["fp16", "bf16"]))
        else:
            tokens = _log(rng, 1, 8192)
            c = _norm("", tokens, 0, 8 * _log(rng, 8, 2048), rng.choice(["fp16", "bf16"]),
                      rng.choice(["none", "same", "same", "fp32"]))
        while work(c)["bytes"] > 8192 * 8192 * 8:
            c["tokens"] //= 2
    elif op == "route":
        experts = _log(rng, 2, 256)
        c = _route("", _log(rng, 1, 8192), experts, rng.randint(1, min(8, experts)), rng.choice(["fp16", "bf16", "fp32"]),
                   rng.random() < 0.5, rng.random() < 0.3)
    else:
        experts = rng.choice([4, 8, 16, 32, 60, 64, 128])
        k = rng.randint(1, min(8, experts))
        hidden = group * _log(rng, 256 // group, 4096 // group)
        inner = group * _log(rng, 1, 14336 // group)
        while 3 * experts * hidden * inner > 3 * 8 * 4096 * 14336:
            inner = group * max(1, inner // (2 * group))
        tokens = rng.choice([_log(rng, 1, 64), _log(rng, 1, 2048)])
        while tokens * k * hidden * inner > 2048 * 6 * 2048 * 1408:
            tokens //= 2
        c = _experts("", max(1, tokens), experts, k, hidden, inner, group,
                     rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]), rng.random() < 0.5, rng.choice([0.0, 0.5, 1.0]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------ inputs

def _pattern(case):
    """Chosen experts [tokens, k]: who shares an expert with whom is part of the case, the same for every
    seed (the seed permutes the experts)."""
    r = random.Random("%s %s %s %s" % (case["tokens"], case["experts"], case["k"], case["skew"]))
    gen = torch.Generator().manual_seed(r.getrandbits(40))
    liking = torch.randn(case["experts"], generator=gen) * case["skew"]
    scores = torch.randn(case["tokens"], case["experts"], generator=gen) + liking
    return scores.topk(case["k"], dim=1).indices


def _words(gen, *sizes):
    return torch.randint(-(1 << 31), 1 << 31, sizes, dtype=torch.int32, device="cuda", generator=gen)


def _scales(gen, k, *sizes):
    """Scales that bring products of inputs of unit size to unit size."""
    spread = 0.2 + 1.6 * torch.rand(*sizes, device="cuda", generator=gen)
    return (spread * (1 / (4.6 * math.sqrt(k)))).half()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)      # noqa: E731
    s = {"case": case}
    if case["op"] == "linear":
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        out = n // 2 if case["gated"] else n
        s.update(words=_words(gen, n * k // 8), scales=_scales(gen, k, k // g, n), x=rand(m, k).half(),
                 bias=(0.5 * rand(n)).half() if case["bias"] else None,
                 residual=(2 * rand(m, out)).half() if case["residual"] else None)
    elif case["op"] == "norm":
        t, d, dtype = case["tokens"], case["dim"], _DTYPES[case["dtype"]]
        if case["heads"]:       # the queries of a fused projection: a view between other heads
            s["x"] = (2 * rand(t, case["heads"] + 4, d)).to(dtype)[:, :case["heads"]]
        else:
            s["x"] = rand(t, d).to(dtype)
        s["weight"] = (1 + 0.2 * rand(d)).to(dtype)
        s["residual"] = None
        if case["residual"] != "none":
            s["residual"] = (4 * rand(t, d)).to(dtype if case["residual"] == "same" else torch.float32)
    elif case["op"] == "route":
        logits = rand(case["tokens"], case["experts"])
        if case["masked"]:      # experts that a token may not use
            logits = logits.masked_fill(torch.rand(logits.shape, device="cuda", generator=gen) < 0.2, -math.inf)
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
    else:
        e, h, i, g = case["experts"], case["hidden"], case["inner"], case["group"]
        label = torch.randperm(e, generator=torch.Generator().manual_seed(seed))
        s.update(x=rand(case["tokens"], h).half(),
                 gate_up=(_words(gen, e, 2 * i * h // 8), _scales(gen, h, e, h // g, 2 * i)),
                 down=(_words(gen, e, h * i // 8), _scales(gen, i, e, i // g, h)),
                 experts=label[_pattern(case)].to("cuda", torch.int32),
                 weights=torch.softmax(rand(case["tokens"], case["k"]), -1),
                 residual=(2 * rand(case["tokens"], h)).half() if case["residual"] else None)
    return s


# ------------------------------------------------------------------------------ the operators

_ACTIVATIONS = {
    "none": lambda z: z,
    "relu": lambda z: z.clamp_min(0),
    "silu": lambda z: z / (1 + torch.exp(-z)),
    "gelu": lambda z: 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5))),
    "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))),
}


def _codes(words, n, k):
    """int32 [n, k] of code - 8 from packed words."""
    shift = torch.arange(0, 32, 4, dtype=torch.int32, device=words.device)
    nibble = ((words.view(n // 16, k // 64, 8, 4, 4, 1) >> shift) & 15) - 8          # [nb, kc, g, t, s, nibble]
    nibble = nibble.view(n // 16, k // 64, 8, 4, 4, 2, 2, 2)                          # nibble: h, b, a
    return nibble.permute(0, 7, 2, 1, 4, 6, 3, 5).reshape(n, k)


def _weight(words, scales, k):
    """fp32 [n, k] from packed words and fp16 scales [k / group, n]."""
    n = scales.shape[1]
    grouped = _codes(words, n, k).float().view(n, scales.shape[0], -1)
    return (grouped * scales.float().t()[:, :, None]).view(n, k)


def _gate(z, activation):
    """act(gate) * up of rows that alternate in runs of eight."""
    z = z.view(z.shape[0], -1, 2, 8)
    return (_ACTIVATIONS[activation](z[:, :, 0]) * z[:, :, 1]).reshape(z.shape[0], -1)


def _plain_linear(s):
    case = s["case"]
    x = s["x"]
    z = x.float() @ _weight(s["words"], s["scales"], x.shape[1]).half().float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _gate(z, case["activation"]) if case["gated"] else _ACTIVATIONS[case["activation"]](z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.half()


def _plain_norm(s, eps=1e-5):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * s["weight"].float()
    y = y.to(s["x"].dtype)
    return y if s["residual"] is None else (y, h.to(s["residual"].dtype))


def _plain_route(s):
    case = s["case"]
    top, index = s["logits"].float().sort(dim=1, descending=True, stable=True)
    top, index = top[:, :case["k"]], index[:, :case["k"]]
    largest = top[:, :1].clamp_min(-3e38)                 # a token without any expert: all weights 0
    p = torch.exp(top - largest)
    total = p.sum(1, keepdim=True) if case["renormalize"] else torch.exp(s["logits"].float() - largest).sum(1, keepdim=True)
    return p / total.clamp_min(1e-30), index.masked_fill(top == -math.inf, -1).int()


def _plain_experts(s):
    case = s["case"]
    x, experts, weights = s["x"].float(), s["experts"].long(), s["weights"]
    hidden, inner, act = case["hidden"], case["inner"], case["activation"]
    y = torch.zeros_like(x) if s["residual"] is None else s["residual"].float()

    def pass_through(rows, e):      # e: an index of one expert, on the device or not
        gate_up = _weight(s["gate_up"][0][e], s["gate_up"][1][e], hidden)
        return _gate(rows @ gate_up.t(), act) @ _weight(s["down"][0][e], s["down"][1][e], inner).t()

    if experts.numel() <= case["experts"]:      # few tokens: the chosen experts, one after the other
        for t in range(case["tokens"]):
            for j in range(case["k"]):
                y[t] += weights[t, j] * pass_through(x[t:t + 1], experts[t, j])[0]
    else:                                       # every expert for every token, with its weight there
        for e in range(case["experts"]):
            y = y + pass_through(x, e) * (weights * (experts == e)).sum(1, keepdim=True)
    return y.half()


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"linear": _plain_linear, "norm": _plain_norm, "route": _plain_route, "experts": _plain_experts}[op](state)
    f = _framework()
    if op == "linear":
        return f.w4a16_linear(state["words"], state["x"], state["scales"], bias=state["bias"],
                              activation=case["activation"], gated=case["gated"], residual=state["residual"])
    if op == "norm":
        return f.rms_norm(state["x"], state["weight"], 1e-5, residual=state["residual"])
    if op == "route":
        return f.moe_route(state["logits"], case["k"], renormalize=case["renormalize"])
    return f.moe_experts(state["x"], state["gate_up"], state["down"], state["experts"], state["weights"],
                         activation=case["activation"], residual=state["residual"])


# ------------------------------------------------------------------------------ bytes, operations, exact values

def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        out = n // 2 if case["gated"] else n
        return {"bytes": n * k // 2 + 2 * n * (k // case["group"]) + 2 * m * k + 2 * m * out * (2 if case["residual"] else 1)
                + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["op"] == "norm":
        values = case["tokens"] * max(1, case["heads"]) * case["dim"]
        b = _BYTES[case["dtype"]]
        extra = {"none": 0, "same": 2 * b, "fp32": 8}[case["residual"]]
        return {"bytes": values * (2 * b + extra) + b * case["dim"], "flops": 5 * values}
    if case["op"] == "route":
        values = case["tokens"] * case["experts"]
        return {"bytes": values * _BYTES[case["dtype"]] + 8 * case["tokens"] * case["k"], "flops": values * (3 + case["k"])}
    touched = int(_pattern(case).unique().numel())
    h, i, t = case["hidden"], case["inner"], case["tokens"]
    weights = 3 * h * i // 2 + 2 * (2 * i * (h // case["group"]) + h * (i // case["group"]))
    return {"bytes": touched * weights + 2 * t * h * (3 if case["residual"] else 2) + 8 * t * case["k"],
            "flops": 6 * t * case["k"] * h * i}


def _exact_weight(words, scales, k, rounded):
    """fp64 [n, k], nibble by nibble."""
    n = scales.shape[1]
    w = words.view(n // 16, k // 64, 32, 4)
    lane = torch.arange(32, device=words.device)
    out = torch.empty(n // 16, 16, k // 64, 64, dtype=torch.float64, device=words.device)
    for nibble in range(8):
        h, b, a = nibble >> 2, nibble >> 1 & 1, nibble & 1
        code = (w >> (4 * nibble) & 15).double() - 8                                 # [nb, kc, lane, s]
        for s in range(4):
            out[:, lane // 4 + 8 * a, :, 16 * s + 2 * (lane % 4) + 8 * b + h] = code[..., s].permute(2, 0, 1)
    out = out.view(n, k) * scales.double().repeat_interleave(k // scales.shape[0], 0).t()
    return out.half().double() if rounded else out


def _exact_activation(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def _exact_gate(z, name):
    column = torch.arange(z.shape[1] // 2, device=z.device)
    gate = 16 * (column // 8) + column % 8
    return _exact_activation(z[:, gate], name) * z[:, gate + 8]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        z = s["x"].double() @ _exact_weight(s["words"], s["scales"], case["k"], True).t()
        if s["bias"] is not None:
            z += s["bias"].double()
        y = _exact_gate(z, case["activation"]) if case["gated"] else _exact_activation(z, case["activation"])
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        y = s["weight"].double() * h * torch.rsqrt(h.square().sum(-1, keepdim=True) / case["dim"] + 1e-5)
        return y if s["residual"] is None else (y, h)
    if case["op"] == "route":
        l = s["logits"].double().cpu()
        p = torch.softmax(l, 1).nan_to_num(0.0)
        chosen = torch.full((case["tokens"], case["k"]), -1, dtype=torch.int32)
        weights = torch.zeros(case["tokens"], case["k"], dtype=torch.float64)
        for t, row in enumerate(l.tolist()):
            best = sorted(range(case["experts"]), key=lambda e: -row[e])[:case["k"]]      # a stable sort
            for j, e in enumerate(best):
                if row[e] > -math.inf:
                    chosen[t, j], weights[t, j] = e, p[t, e]
        if case["renormalize"]:
            weights = weights / weights.sum(1, keepdim=True).clamp_min(1e-300)
        return weights, chosen
    y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, slot = (s["experts"] == e).nonzero(as_tuple=True)
        if token.numel():
            inner = _exact_gate(s["x"][token].double() @ _exact_weight(s["gate_up"][0][e], s["gate_up"][1][e], case["hidden"],
                                                                       False).t(), case["activation"])
            out = inner @ _exact_weight(s["down"][0][e], s["down"][1][e], case["inner"], False).t()
            y.index_add_(0, token, out * s["weights"][token, slot, None].double())
    return y if s["residual"] is None else y + s["residual"].double()
