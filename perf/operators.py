"""Measured cases of the gated feed-forward block and of the microscaled 4-bit linear layers.

Three operators of the encoders' packed token rows:

* ``ffn``: ``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual`` in bf16, forward, or forward and
  backward (gradients of x, the weights, the biases and the residual);
* ``quantize``: a matrix rounded to microscaled 4-bit floating point (MXFP4: a power-of-two scale per 32
  values; NVFP4: an E4M3 scale per 16 values and a power-of-two scale per row), returned as the values that
  the codes stand for;
* ``linear``: ``y = Q(x) Q(W)^T + b + residual`` with both operands held in 4 bits (the weight is quantised
  once, before the call), forward, or forward and the input gradient ``dx = dy Q(W)``;
* ``ffn4``: the gated block over 4-bit operands, ``h = act(Q(x) Q(Wg)^T) * (Q(x) Q(Wu)^T)``,
  ``y = Q(h) Q(Wd)^T + residual``.

``own`` false computes the plain form in 32 bits, ``own`` true calls the framework.
"""

import math

import torch

own = False

E2M1_MAX = 6.0
E4M3_MAX = 448.0
ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "quick_gelu")


# ------------------------------------------------------------------- cases
def listed():
    def ffn(name, t, h, i, act, bias, train):
        return {"name": name, "op": "ffn", "t": t, "h": h, "i": i, "act": act, "bias": bias, "train": train}

    def quant(name, r, c, fmt, dtype):
        return {"name": name, "op": "quantize", "r": r, "c": c, "fmt": fmt, "dtype": dtype}

    def linear(name, m, n, k, fmt, bias, grad):
        return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "fmt": fmt, "bias": bias, "grad": grad}

    return [
        # one token through a decoder layer's block: the last-token step of an online query
        ffn("ffn-1-token", 1, 2048, 6144, "silu", False, False),
        # one short query through an encoder layer of the text-image retriever
        ffn("ffn-23-tokens", 23, 768, 1152, "gelu", False, False),
        # a packed batch of documents, indexing (no gradients)
        ffn("ffn-documents", 12289, 2048, 6144, "silu", False, False),
        # a ragged training chunk of the text-image retriever
        ffn("ffn-train-ragged", 1111, 768, 1152, "gelu", False, True),
        # a vision tower's block with biases, an odd number of patches
        ffn("ffn-train-bias", 2047, 1280, 3416, "silu", True, True),
        # a full training chunk of the decoder embedder
        ffn("ffn-train-chunk", 8192, 2048, 6144, "silu", False, True),
        # the activations of one short query on their way into a 4-bit layer
        quant("quantize-query", 37, 2048, "mxfp4", "bfloat16"),
        # a weight matrix from its fp32 master copy, an odd number of rows
        quant("quantize-weight", 12283, 2048, "nvfp4", "float32"),
        # one token through the fused gate / up projection
        linear("linear4-1-token", 1, 12288, 2048, "nvfp4", False, False),
        # a ragged batch with a contraction that ends inside a block, and its input gradient
        linear("linear4-grad-odd", 1531, 1544, 1000, "mxfp4", True, True),
        # a packed batch of documents through a down projection
        linear("linear4-documents", 8192, 2048, 6144, "nvfp4", False, False),
        # the whole block in 4 bits on a packed batch
        {"name": "ffn4-documents", "op": "ffn4", "t": 8192, "h": 2048, "i": 6144, "act": "silu", "fmt": "mxfp4"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high, step):
    """A width that is a multiple of ``step``, logarithmically spread, never one of the excluded sizes."""

    while True:
        w = max(step, _log_int(rng, low, high) // step * step)
        if w not in (1536, 3072):
            return w


def draw(rng):
    op = rng.choice(("ffn", "ffn", "quantize", "linear", "linear", "ffn4"))
    if op == "ffn":
        return {"op": op, "t": _log_int(rng, 1, 8191), "h": _width(rng, 64, 2048, 8), "i": _width(rng, 64, 6144, 8),
                "act": rng.choice(ACTIVATIONS), "bias": rng.random() < 0.4, "train": rng.random() < 0.5}
    if op == "quantize":
        return {"op": op, "r": _log_int(rng, 1, 12283), "c": _log_int(rng, 17, 6144), "fmt": rng.choice(("mxfp4", "nvfp4")),
                "dtype": rng.choice(("bfloat16", "float16", "float32"))}
    if op == "linear":
        grad = rng.random() < 0.3
        return {"op": op, "m": _log_int(rng, 1, 8191), "n": _width(rng, 64, 12288, 8) if grad else _log_int(rng, 33, 12289),
                "k": _width(rng, 64, 6144, 8) if grad else _log_int(rng, 33, 6144), "fmt": rng.choice(("mxfp4", "nvfp4")),
                "bias": rng.random() < 0.4, "grad": grad}
    return {"op": op, "t": _log_int(rng, 1, 8191), "h": _width(rng, 64, 2048, 8), "i": _width(rng, 64, 6144, 8),
            "act": rng.choice(ACTIVATIONS), "fmt": "mxfp4"}


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """The case's inputs, from the seed alone."""

    gen = torch.Generator("cuda").manual_seed(1_000_003 * int(seed) + 17)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    op = case["op"]
    if op in ("ffn", "ffn4"):
        t, h, i = case["t"], case["h"], case["i"]
        # rows as they leave a norm: unit scale with a gain per channel
        gain = 0.5 + torch.rand(h, generator=gen, device="cuda")
        d = {"x": (torch.randn(t, h, generator=gen, device="cuda") * gain).to(torch.bfloat16),
             "gate_up": normal(2 * i, h, std=h ** -0.5), "down": normal(h, i, std=i ** -0.5), "residual": normal(t, h)}
        if case.get("bias"):
            d["gate_up_bias"], d["down_bias"] = normal(2 * i, std=0.1), normal(h, std=0.1)
        if case.get("train"):
            d["dy"] = normal(t, h, std=0.01)
        return d
    if op == "quantize":
        # rows and columns of different magnitudes, as activations and weights have
        rows = torch.exp(torch.randn(case["r"], 1, generator=gen, device="cuda"))
        cols = 0.5 + torch.rand(case["c"], generator=gen, device="cuda")
        x = torch.randn(case["r"], case["c"], generator=gen, device="cuda") * rows * cols
        return {"x": x.to(getattr(torch, case["dtype"]))}
    m, n, k = case["m"], case["n"], case["k"]
    d = {"x": normal(m, k), "weight": normal(n, k, std=k ** -0.5), "residual": normal(m, n)}
    if case["bias"]:
        d["bias"] = normal(n, std=0.1)
    if case["grad"]:
        d["dy"] = normal(m, n, std=0.01)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    op = case["op"]
    if op == "ffn" and case["train"] and own:
        for name in ("x", "gate_up", "down", "residual", "gate_up_bias", "down_bias"):
            if name in d:
                d[name].requires_grad_()
    if op in ("linear", "ffn4"):  # the weights are quantised once and kept
        names = ("weight",) if op == "linear" else ("gate_up", "down")
        if own:
            from representax_b200.ops.fp4 import quantize

            # the fused projection keeps its gate and up rows as two parts
            d.update({name: quantize(d[name], case["fmt"], parts=2 if name == "gate_up" else 1) for name in names})
            if op == "linear" and case["grad"]:
                d["x"].requires_grad_()
        else:
            d.update({name: _fake_quantize(d[name], case["fmt"]) for name in names})
    d["case"] = dict(case)
    return d


# ------------------------------------------------------------- plain forms
def _round_e2m1(v):
    """Nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), larger values to 6."""

    a = v.abs().clamp(max=E2M1_MAX)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(a / step) * step * torch.sign(v)


def _fake_quantize(x, fmt):
    """The fp32 values that the 4-bit codes and scales of ``x`` (rows x columns) stand for."""

    xf = x.float()
    r, c = xf.shape
    block = 32 if fmt == "mxfp4" else 16
    pad = -c % block
    b = torch.nn.functional.pad(xf, (0, pad)).reshape(r, (c + pad) // block, block)
    amax = b.abs().amax(-1, keepdim=True)
    # divisors are tensors: a division by a Python number may be computed as a product with its rounded inverse
    six = torch.full_like(amax, E2M1_MAX)
    if fmt == "mxfp4":
        scale = _pow2_ceil(amax / six)
    else:
        row = _pow2_ceil(amax.amax(1, keepdim=True) / (six[:, :1] * E4M3_MAX))
        scale = (amax / six / row).clamp(max=E4M3_MAX).to(torch.float8_e4m3fn).float() * row
    q = torch.where(scale > 0, _round_e2m1(b / torch.where(scale > 0, scale, 1.0)) * scale, 0.0)
    return q.reshape(r, c + pad)[:, :c].contiguous()


def _pow2_ceil(v):
    """2^ceil(log2 v) for v > 0 (at least 2^-126), 1 for v = 0."""

    mantissa, exponent = torch.frexp(v)
    e = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(min=-126)
    return torch.where(v > 0, torch.ldexp(torch.ones_like(v), e), 1.0)


def _act(g, name):
    """Activation and its derivative in 32 bits."""

    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "quick_gelu":
        s = 1 / (1 + torch.exp(-1.702 * g))
        return g * s, s * (1 + 1.702 * g * (1 - s))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * 0.044715 * g * g)


def _plain_ffn(s, case):
    x, wgu, wd, res = (s[k].float() for k in ("x", "gate_up", "down", "residual"))
    i = case["i"]
    z = x @ wgu.T
    if case["bias"]:
        z = z + s["gate_up_bias"].float()
    a, da = _act(z[:, :i], case["act"])
    u = z[:, i:]
    h = a * u
    y = h @ wd.T + res
    if case["bias"]:
        y = y + s["down_bias"].float()
    out = {"y": y.to(torch.bfloat16)}
    if case["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        dz = torch.cat([dh * u * da, dh * a], 1)
        grads = {"dx": dz @ wgu, "dgate_up": dz.T @ x, "ddown": dy.T @ h, "dresidual": dy}
        if case["bias"]:
            grads["dgate_up_bias"], grads["ddown_bias"] = dz.sum(0), dy.sum(0)
        out.update({k: v.to(torch.bfloat16) for k, v in grads.items()})
    return out


def _plain_linear(s, case):
    y = _fake_quantize(s["x"], case["fmt"]) @ s["weight"].T + s["residual"].float()
    if case["bias"]:
        y = y + s["bias"].float()
    out = {"y": y.to(torch.bfloat16)}
    if case["grad"]:
        out["dx"] = (s["dy"].float() @ s["weight"]).to(torch.bfloat16)
    return out


def _plain_ffn4(s, case):
    i = case["i"]
    z = _fake_quantize(s["x"], case["fmt"]) @ s["gate_up"].T
    h = _act(z[:, :i], case["act"])[0] * z[:, i:]
    return {"y": (_fake_quantize(h, case["fmt"]) @ s["down"].T + s["residual"].float()).to(torch.bfloat16)}


# --------------------------------------------------------------------- run
def _own_ffn(s, case):
    from representax_b200.ops.ffn import gated_feed_forward

    y = gated_feed_forward(s["x"], s["gate_up"], s["down"], activation=case["act"],
                           gate_up_bias=s.get("gate_up_bias"), down_bias=s.get("down_bias"), residual=s["residual"])
    out = {"y": y}
    if case["train"]:
        names = ["x", "gate_up", "down", "residual"] + (["gate_up_bias", "down_bias"] if case["bias"] else [])
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return out


def _own_linear(s, case):
    from representax_b200.ops.fp4 import linear_fp4

    y = linear_fp4(s["x"], s["weight"], s.get("bias"), s["residual"])
    out = {"y": y}
    if case["grad"]:
        out["dx"] = torch.autograd.grad(y, s["x"], s["dy"])[0]
    return out


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        if op == "quantize":
            return {"values": _fake_quantize(state["x"], case["fmt"])}
        return {"ffn": _plain_ffn, "linear": _plain_linear, "ffn4": _plain_ffn4}[op](state, case)
    if op == "quantize":
        from representax_b200.ops.fp4 import dequantize, quantize

        return {"values": dequantize(quantize(state["x"], case["fmt"]), torch.float32)}
    if op == "ffn4":
        from representax_b200.ops.fp4 import gated_feed_forward_fp4

        return {"y": gated_feed_forward_fp4(state["x"], state["gate_up"], state["down"], activation=case["act"],
                                            residual=state["residual"])}
    return {"ffn": _own_ffn, "linear": _own_linear}[op](state, case)


# -------------------------------------------------------------------- work
def _bytes4(rows, k, fmt):
    """Bytes of a matrix held in 4 bits with its scales."""

    return rows * k / 2 + rows * -(-k // (32 if fmt == "mxfp4" else 16)) + (4 * rows if fmt == "nvfp4" else 0)


def work(case):
    op = case["op"]
    if op == "quantize":
        size = {"float32": 4}.get(case["dtype"], 2)
        return {"bytes": case["r"] * case["c"] * (size + 4), "flops": 4 * case["r"] * case["c"]}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        passes = 2 if case["grad"] else 1
        return {"bytes": 2 * m * k * passes + _bytes4(n, k, case["fmt"]) + 2 * m * n * (2 + (passes - 1)),
                "flops": 2 * m * n * k * passes}
    t, h, i = case["t"], case["h"], case["i"]
    if op == "ffn4":
        return {"bytes": 6 * t * h + _bytes4(2 * i, h, case["fmt"]) + _bytes4(h, i, case["fmt"]), "flops": 6 * t * h * i}
    weights = 2 * 3 * h * i
    if case["train"]:  # x, residual, dy, the weights in; y, three gradients of rows, the weights' gradients out
        return {"bytes": 2 * weights + 2 * t * h * 6, "flops": 18 * t * h * i}
    return {"bytes": weights + 2 * t * h * 3, "flops": 6 * t * h * i}


# ------------------------------------------------------------------- exact
def _exact_quantize(x, fmt):
    """The formats' definition in 64 bits: nearest grid values found by their midpoints."""

    x = x.double()
    r, c = x.shape
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    size = 32 if fmt == "mxfp4" else 16
    blocks = -(-c // size)
    padded = torch.zeros(r, blocks * size, dtype=torch.float64, device=x.device)
    padded[:, :c] = x
    v = padded.view(r, blocks, size)
    top = v.abs().max(dim=2).values

    def up_to_power(t):
        e = torch.ceil(torch.log2(t.clamp(min=1e-300)))
        e = torch.where(torch.exp2(e) < t, e + 1, torch.where(torch.exp2(e - 1) >= t, e - 1, e))
        return torch.where(t > 0, torch.exp2(e.clamp(min=-126)), torch.ones_like(t))

    if fmt == "mxfp4":
        scale = up_to_power(top / 6)
    else:
        row = up_to_power(top.max(dim=1, keepdim=True).values / (6 * 448))
        want = (top / 6 / row).clamp(max=448)
        # E4M3: steps of 2^(e - 3), e at least -6
        e = torch.floor(torch.log2(want.clamp(min=2.0 ** -6)))
        e = torch.where(torch.exp2(e + 1) <= want, e + 1, torch.where(torch.exp2(e) > want.clamp(min=2.0 ** -6), e - 1, e))
        unit = torch.exp2(e - 3)
        scale = torch.round(want / unit) * unit * row
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    m = v.abs() / safe[..., None]
    edges = (grid[1:] + grid[:-1]) / 2
    low = torch.bucketize(m, edges)               # a value on an edge stays below it ...
    high = torch.bucketize(m, edges, right=True)  # ... or goes above it
    code = torch.where(low % 2 == 0, low, high)   # ties to the even code
    q = grid[code] * torch.sign(v) * torch.where(scale > 0, scale, torch.zeros_like(scale))[..., None]
    return q.view(r, blocks * size)[:, :c]


def _exact_act(g, name):
    """Activation and derivative in 64 bits."""

    if name in ("silu", "quick_gelu"):
        k = 1.0 if name == "silu" else 1.702
        s = torch.sigmoid(k * g)
        return g * s, s + k * g * s * torch.sigmoid(-k * g)
    if name == "gelu":
        half = torch.special.ndtr(g)
        return g * half, half + g * torch.exp(-g.square() / 2) * (2 * math.pi) ** -0.5
    inner = (2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)
    slope = (2 / math.pi) ** 0.5 * (1 + 3 * 0.044715 * g ** 2)
    return g * torch.sigmoid(2 * inner), torch.sigmoid(2 * inner) + 2 * g * slope * torch.sigmoid(2 * inner) * torch.sigmoid(-2 * inner)


def exact(case, seed):
    d = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        return {"values": _exact_quantize(d["x"], case["fmt"])}
    if op == "linear":
        w = _exact_quantize(d["weight"], case["fmt"])
        y = torch.matmul(_exact_quantize(d["x"], case["fmt"]), w.t()) + d["residual"].double()
        out = {"y": y + d["bias"].double() if case["bias"] else y}
        if case["grad"]:
            out["dx"] = torch.matmul(d["dy"].double(), w)
        return out
    i = case["i"]
    if op == "ffn4":
        w1, w2 = _exact_quantize(d["gate_up"], case["fmt"]), _exact_quantize(d["down"], case["fmt"])
        z = torch.matmul(_exact_quantize(d["x"], case["fmt"]), w1.t())
        hidden = _exact_act(z[:, :i], case["act"])[0] * z[:, i:]
        return {"y": torch.matmul(_exact_quantize(hidden, case["fmt"]), w2.t()) + d["residual"].double()}
    f = {k: v.double() for k, v in d.items()}
    gate, up = torch.matmul(f["x"], f["gate_up"][:i].t()), torch.matmul(f["x"], f["gate_up"][i:].t())
    if case["bias"]:
        gate, up = gate + f["gate_up_bias"][:i], up + f["gate_up_bias"][i:]
    a, slope = _exact_act(gate, case["act"])
    out = {"y": torch.matmul(a * up, f["down"].t()) + f["residual"]}
    if case["bias"]:
        out["y"] = out["y"] + f["down_bias"]
    if case["train"]:
        dy = f["dy"]
        dh = torch.matmul(dy, f["down"])
        dgate, dup = dh * up * slope, dh * a
        out["dx"] = torch.matmul(dgate, f["gate_up"][:i]) + torch.matmul(dup, f["gate_up"][i:])
        out["dgate_up"] = torch.cat([torch.matmul(dgate.t(), f["x"]), torch.matmul(dup.t(), f["x"])])
        out["ddown"] = torch.matmul(dy.t(), a * up)
        out["dresidual"] = dy
        if case["bias"]:
            out["dgate_up_bias"], out["ddown_bias"] = torch.cat([dgate.sum(0), dup.sum(0)]), dy.sum(0)
    return out
