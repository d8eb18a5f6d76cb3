"""Gated feed-forward kernels against the formula in 64 bits.

Tolerances (2-norm of the difference over the 2-norm of the result): the
kernels round to bf16 twice on the way to y (h, y), to a gradient of rows or
weights (dz or h, the gradient itself), each by at most 2^-9 of a value; what
the backward keeps is rounded to 11 bits. Two roundings give 2^-8; products
accumulate in fp32, far below that.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -8
ACTS = ("silu", "gelu", "gelu_tanh", "quick_gelu")


def _dev():
    return torch.device("cuda", 0)


def _status_ok():
    from representax_b200.ops._ext import check_status

    torch.cuda.synchronize()
    check_status(_dev())


def _rel(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm().clamp_min(1e-300))


def _act(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "quick_gelu":
        return g * torch.sigmoid(1.702 * g)
    if name == "gelu":
        return g * torch.special.ndtr(g)
    return 0.5 * g * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)))


def _formula(x, w1, w2, act, b1=None, b2=None, res=None):
    z = x @ w1.T
    z = z if b1 is None else z + b1
    i = w2.shape[1]
    y = (_act(z[:, :i], act) * z[:, i:]) @ w2.T
    y = y if b2 is None else y + b2
    return y if res is None else y + res


def _operands(t, h, i, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(1000 * t + h + i + seed)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=_dev()) * std).to(torch.bfloat16)  # noqa: E731
    ops = {"x": n(t, h), "w1": n(2 * i, h, std=h ** -0.5), "w2": n(h, i, std=i ** -0.5),
           "b1": n(2 * i, std=0.2) if bias else None, "b2": n(h, std=0.2) if bias else None, "res": n(t, h)}
    return ops, n(t, h)


def _run(o, act):
    from representax_b200.ops.ffn import gated_feed_forward

    return gated_feed_forward(o["x"], o["w1"], o["w2"], activation=act, gate_up_bias=o["b1"], down_bias=o["b2"],
                              residual=o["res"])


def _want(o, act):
    f = {k: None if v is None else v.detach().double() for k, v in o.items()}
    return _formula(f["x"], f["w1"], f["w2"], act, f["b1"], f["b2"], f["res"])


SIZES = [(1, 64, 64), (1, 2048, 512), (5, 8, 8), (15, 72, 200), (16, 128, 128), (17, 96, 136), (32, 256, 264), (33, 256, 264),
         (64, 512, 384), (65, 120, 1000), (128, 264, 256), (129, 1024, 64), (255, 64, 520), (256, 256, 128), (257, 776, 1152),
         (700, 2048, 128)]


@pytest.mark.parametrize("t,h,i", SIZES)
@pytest.mark.parametrize("bias", [False, True])
def test_forward(t, h, i, bias):
    o, _ = _operands(t, h, i, bias=bias)
    if t % 2:
        o["res"] = None
    act = ACTS[(t + i // 8) % 4]
    y = _run(o, act)
    _status_ok()
    assert _rel(y, _want(o, act)) < TOL


@pytest.mark.parametrize("t,h,i", [(32, 64, 2568), (33, 64, 2560), (33, 64, 2568), (64, 72, 2560), (64, 136, 1000), (65, 64, 2560),
                                   (65, 200, 520), (200, 200, 1600), (600, 200, 1600), (600, 264, 1600), (2000, 256, 1600),
                                   (300, 776, 2504)])
def test_forward_on_both_sides_of_the_few_row_bounds(t, h, i):
    o, _ = _operands(t, h, i)
    y = _run(o, "silu")
    _status_ok()
    assert _rel(y, _want(o, "silu")) < TOL
    assert max(_rel(y[r:r + 16], _want(o, "silu")[r:r + 16]) for r in range(0, t, 16)) < 2 * TOL


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [3, 70])
def test_activations(act, t):
    o, _ = _operands(t, 64, 96)
    o["x"] = o["x"] * 4  # both tails of the activation
    y = _run(o, act)
    _status_ok()
    assert _rel(y, _want(o, act)) < TOL


def _between(got, want, error):
    """Rounding keeps the order, so got lies between the roundings of want - error and want + error."""

    low, high = (want - error).to(torch.bfloat16), (want + error).to(torch.bfloat16)
    assert got.dtype == torch.bfloat16 and bool(((got >= low) & (got <= high)).all())


def _act_grad(g, name):
    g = g.clone().requires_grad_()
    if name == "gelu":  # Phi by its complement: exact in the lower tail
        value = g * 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
    elif name == "gelu_tanh":
        value = g * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))
    else:
        value = g * torch.sigmoid((1.702 if name == "quick_gelu" else 1.0) * g)
    (grad,) = torch.autograd.grad(value.sum(), g)
    return value.detach(), grad


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [1, 40, 300])
def test_activation_value_by_value(act, t):
    """act(g) and act'(g) of 512 gates from -8 to 8, each between the bf16 roundings of the ends of its interval. The
    block is built so that y is h itself (u one, the down projection the identity) and the gate bias's gradient of one
    row is dz. Before that rounding the activation is off by 2e-5 of itself, the kept factors by 2^-11 more (11
    bits), and act' next to its zero by the absolute error of its parts, below 2e-6 there."""

    from representax_b200.ops.ffn import gated_feed_forward

    n = 512
    gates = torch.linspace(-8, 8, n, device=_dev()).to(torch.bfloat16)
    x = torch.zeros(t, n, dtype=torch.bfloat16, device=_dev())
    x[:, 0] = 1
    w1 = torch.zeros(2 * n, n, dtype=torch.bfloat16, device=_dev())
    w1[:n, 0], w1[n:, 0] = gates, 1
    w2 = torch.eye(n, dtype=torch.bfloat16, device=_dev())
    value, grad = _act_grad(gates.double(), act)
    _between(gated_feed_forward(x, w1, w2, activation=act), value, 2e-5 * value.abs())
    b1 = torch.zeros(2 * n, dtype=torch.bfloat16, device=_dev(), requires_grad=True)
    y = gated_feed_forward(x, w1, w2, activation=act, gate_up_bias=b1)
    _between(y, value, 2e-5 * value.abs())
    dy = torch.zeros_like(y)
    dy[t - 1] = 1
    (db,) = torch.autograd.grad(y, b1, dy)
    _status_ok()
    _between(db[:n], grad, (2.0 ** -11 + 2e-5) * grad.abs() + 2e-6 * (grad.abs() < 0.05))
    _between(db[n:], value, (2.0 ** -11 + 2e-5) * value.abs())


@pytest.mark.parametrize("t,h,i", [(1, 64, 64), (7, 96, 200), (33, 128, 72), (64, 512, 384), (257, 264, 1000), (513, 768, 1152)])
@pytest.mark.parametrize("act", ACTS)
def test_gradients(t, h, i, act):
    o, dy = _operands(t, h, i)
    leaves = {k: v.requires_grad_() for k, v in o.items()}
    grads = torch.autograd.grad(_run(leaves, act), list(leaves.values()), dy)
    _status_ok()
    ref = {k: v.detach().double().requires_grad_() for k, v in o.items()}
    want = torch.autograd.grad(_formula(ref["x"], ref["w1"], ref["w2"], act, ref["b1"], ref["b2"], ref["res"]),
                               list(ref.values()), dy.double())
    for name, g, w in zip(leaves, grads, want):
        assert g.dtype == torch.bfloat16 and _rel(g, w) < TOL, name


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """<gradient, direction> against the central difference of the loss in 64 bits (step 1e-4: its error is the
    third derivative's times 1e-8)."""

    o, dy = _operands(40, 64, 96)
    leaves = {k: v.requires_grad_() for k, v in o.items()}
    grads = dict(zip(leaves, torch.autograd.grad(_run(leaves, act), list(leaves.values()), dy)))
    f = {k: v.detach().double() for k, v in o.items()}
    gen = torch.Generator(device="cuda").manual_seed(5)

    def loss(**moved):
        v = {**f, **moved}
        return float((_formula(v["x"], v["w1"], v["w2"], act, v["b1"], v["b2"], v["res"]) * dy.double()).sum())

    for name, g in grads.items():
        # the gradient's own direction (a large signal) and a random one
        for d in (g.double(), torch.randn(g.shape, generator=gen, device=_dev(), dtype=torch.float64)):
            d = d / d.norm()
            diff = (loss(**{name: f[name] + 1e-4 * d}) - loss(**{name: f[name] - 1e-4 * d})) / 2e-4
            assert abs(float((g.double() * d).sum()) - diff) < (TOL + 1e-5) * float(g.double().norm()), name


@pytest.mark.parametrize("need", ["x", "w1", "w2", "b1", "b2", "res"])
def test_single_gradient(need):
    o, dy = _operands(70, 64, 96)
    o[need].requires_grad_()
    (g,) = torch.autograd.grad(_run(o, "silu"), [o[need]], dy)
    ref = {k: v.detach().double() for k, v in o.items()}
    ref[need].requires_grad_()
    (w,) = torch.autograd.grad(_formula(ref["x"], ref["w1"], ref["w2"], "silu", ref["b1"], ref["b2"], ref["res"]), [ref[need]],
                               dy.double())
    assert _rel(g, w) < TOL


def test_gradients_of_spread_magnitudes():
    """What the backward keeps holds blocks of any magnitude (2^-66 to 2^66 here)."""

    o, dy = _operands(64, 128, 64, bias=False)
    o["res"] = None
    # up rows scaled per column group: the kept u act'(g) of neighbouring blocks differ by 2^132
    scale = torch.ones(128, 1, device=_dev())
    scale[64:96] = 2.0 ** 66
    scale[96:] = 2.0 ** -66
    o["w1"] = (o["w1"].float() * scale).to(torch.bfloat16).requires_grad_()
    o["x"].requires_grad_()
    gw, gx = torch.autograd.grad(_run(o, "silu"), [o["w1"], o["x"]], dy)
    r = {k: None if v is None else v.detach().double() for k, v in o.items()}
    r["w1"].requires_grad_()
    r["x"].requires_grad_()
    ww, wx = torch.autograd.grad(_formula(r["x"], r["w1"], r["w2"], "silu"), [r["w1"], r["x"]], dy.double())
    for rows in (slice(0, 32), slice(32, 64), slice(64, 96), slice(96, 128)):
        assert _rel(gw[rows], ww[rows]) < TOL
    assert _rel(gx, wx) < TOL


def test_parameters_with_accumulators():
    """fp32 parameters get fp32 gradients; a main_grad is added into."""

    from representax_b200.ops.ffn import gated_feed_forward

    o, dy = _operands(90, 64, 96, bias=False)
    w1, w2 = (torch.nn.Parameter(o[k].float()) for k in ("w1", "w2"))
    w2.main_grad = torch.ones(w2.shape, device=_dev())
    y = gated_feed_forward(o["x"], w1, w2, activation="silu")
    y.backward(dy)
    r1, r2 = (o[k].double().requires_grad_() for k in ("w1", "w2"))
    want = torch.autograd.grad(_formula(o["x"].double(), r1, r2, "silu"), [r1, r2], dy.double())
    assert w1.grad.dtype == torch.float32 and _rel(w1.grad, want[0]) < TOL
    assert w2.grad is None and _rel(w2.main_grad - 1, want[1]) < TOL


def test_empty_and_odd_widths():
    o, _ = _operands(4, 64, 96)
    o["x"], o["res"] = o["x"][:0], o["res"][:0]
    assert _run(o, "silu").shape == (0, 64)
    o, dy = _operands(9, 60, 84)  # not multiples of 8: the PyTorch statement
    o["x"].requires_grad_()
    y = _run(o, "gelu")
    assert _rel(y.detach(), _want(o, "gelu")) < TOL
    assert torch.autograd.grad(y, o["x"], dy)[0].shape == o["x"].shape


@pytest.mark.parametrize("t", [5, 40, 300])
def test_strided_and_misaligned_operands(t):
    o, dy = _operands(t, 64, 96)
    want = _want(o, "silu")
    wide = torch.zeros(t, 64 + 3, dtype=torch.bfloat16, device=_dev())
    wide[:, 3:] = o["x"]
    flat = torch.zeros(o["w1"].numel() + 1, dtype=torch.bfloat16, device=_dev())
    flat[1:] = o["w1"].reshape(-1)
    bias = torch.zeros(2 * 96 + 1, dtype=torch.bfloat16, device=_dev())
    bias[1:] = o["b1"]
    v = dict(o, x=wide[:, 3:], w1=flat[1:].view(192, 64), w2=o["w2"].T.contiguous().T, b1=bias[1:],
             res=o["res"].T.contiguous().T)
    assert torch.equal(_run(v, "silu"), _run(o, "silu"))
    leaves = [v["x"].requires_grad_(), v["w1"].requires_grad_(), v["w2"].requires_grad_()]
    y = _run(v, "silu")
    assert _rel(y.detach(), want) < TOL
    dy_t = dy.T.contiguous().T
    got = torch.autograd.grad(y, leaves, dy_t)
    plain = [o[k].detach().requires_grad_() for k in ("x", "w1", "w2")]
    ref = torch.autograd.grad(_run(dict(o, x=plain[0], w1=plain[1], w2=plain[2]), "silu"), plain, dy)
    for a, b in zip(got, ref):
        assert _rel(a, b.double()) < TOL
    expanded = o["x"][:1].expand(t, 64)  # one row for all tokens
    assert torch.equal(_run(dict(o, x=expanded), "silu"), _run(dict(o, x=expanded.contiguous()), "silu"))


@pytest.mark.parametrize("t", [6, 50, 300])
def test_nonfinite_rows_stay_rows(t):
    o, dy = _operands(t, 64, 96)
    clean = _run(o, "silu")
    x = o["x"].clone()
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y = _run(dict(o, x=x), "silu")
    keep = [r for r in range(t) if r not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])
    assert y[1].isnan().all() and not y[2].isfinite().any()
    x = x.requires_grad_()
    (g,) = torch.autograd.grad(_run(dict(o, x=x), "silu"), [x], dy)
    assert g[keep].isfinite().all() and g[1].isnan().all()


@pytest.mark.parametrize("t", [1, 40, 300])
def test_other_stream_and_repeats(t):
    o, dy = _operands(t, 256, 264)
    first = _run(o, "silu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [_run(o, "silu") for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(first, a) for a in again)  # no result depends on timing
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _run(o, "silu")
    graph.replay()
    _status_ok()
    assert torch.equal(y, first)


def test_refusals():
    from representax_b200.ops.ffn import gated_feed_forward

    o, _ = _operands(4, 64, 96)
    call = lambda **k: gated_feed_forward(**{**dict(x=o["x"], gate_up=o["w1"], down=o["w2"], activation="silu"), **k})  # noqa: E731
    with pytest.raises(ValueError, match="activation"):
        call(activation="relu6")
    with pytest.raises(ValueError, match="matrices"):
        call(x=o["x"][0])
    with pytest.raises(ValueError, match="gate_up must be"):
        call(gate_up=o["w1"][:-2])
    with pytest.raises(ValueError, match="gate_up must be"):
        call(down=o["w2"][:, :-8])
    with pytest.raises(ValueError, match="gate_up_bias"):
        call(gate_up_bias=o["b2"])
    with pytest.raises(ValueError, match="down_bias"):
        call(down_bias=o["b1"])
    with pytest.raises(ValueError, match="residual"):
        call(residual=o["res"].float())
    with pytest.raises(RuntimeError, match="device"):
        call(down=o["w2"].cpu())


def test_model_layers_agree():
    """A ModernBERT and a Qwen3 tower with the fused blocks against their separate layers: the hidden states
    differ by roundings only (each of 2 layers rounds z once more in the separate form)."""

    from representax_b200.models.qwen3 import Qwen3TextConfig, Qwen3TextTower
    from representax_b200.ops import nn as N

    cfg = Qwen3TextConfig(vocab_size=100, hidden_size=128, intermediate_size=264, num_hidden_layers=2, num_attention_heads=2,
                          num_key_value_heads=2, head_dimension=64)
    tower = Qwen3TextTower(cfg, torch.Generator().manual_seed(0)).to(_dev())
    seg = N.Segments.from_lengths([33, 1, 50], _dev())
    emb = torch.randn(seg.total, 128, device=_dev()).to(torch.bfloat16)
    pos = torch.cat([torch.arange(n) for n in seg.lengths()]).to(_dev())
    with torch.no_grad():
        plain = tower(emb, seg, pos)
        with N.fused_feed_forward():
            fused = tower(emb, seg, pos)
    assert not torch.equal(plain, fused) and _rel(fused, plain) < 4 * TOL
