"""Microscaled 4-bit kernels: the quantiser bit for bit against the PyTorch
statement, products against the same codes multiplied in 64 bits.

Tolerances (2-norm of the difference over the 2-norm of the result): a product
is rounded once to bf16, at most 2^-9 of a value; its fp32 accumulation over K
terms adds at most K 2^-24 of the sum of magnitudes, below 2^-12 for the sizes
here.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -9 + 2.0 ** -12
FMTS = ("mxfp4", "nvfp4")


def _dev():
    return torch.device("cuda", 0)


def _status_ok():
    from representax_b200.ops._ext import check_status

    torch.cuda.synchronize()
    check_status(_dev())


def _rel(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm().clamp_min(1e-300))


def _randn(*shape, seed=0, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=_dev()) * std).to(dtype)


def _same(op, ref):
    assert torch.equal(op.data.cpu(), ref.data)
    assert torch.equal(op.scales.cpu(), ref.scales)
    assert (op.row_scale is None) == (ref.row_scale is None)
    if op.row_scale is not None:
        assert torch.equal(op.row_scale.cpu(), ref.row_scale)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("r,c,parts", [(1, 1, 1), (1, 2048, 1), (3, 17, 1), (37, 83, 1), (300, 1000, 2), (5, 9000, 1),
                                       (129, 33, 1), (130, 64, 2), (256, 256, 1), (2, 1025, 1)])
def test_quantize_matches_statement(fmt, dtype, r, c, parts):
    from representax_b200.ops.fp4 import dequantize, fake_quantize_reference, quantize

    x = (_randn(r, c, seed=r + c, dtype=torch.float32) * torch.exp(_randn(r, 1, seed=c, dtype=torch.float32))).to(dtype)
    op = quantize(x, fmt, parts=parts)
    _same(op, quantize(x.cpu(), fmt, parts=parts))
    want = fake_quantize_reference(x, fmt)
    assert torch.equal(dequantize(op, torch.float32), want)
    assert torch.equal(dequantize(op).float(), want)  # exact in bf16 too
    wide = torch.full((r, c + 5), -1.0, device=_dev())
    dequantize(op, out=wide[:, 2:c + 2])
    assert torch.equal(wide[:, 2:c + 2], want) and bool((wide[:, :2] == -1).all()) and bool((wide[:, c + 2:] == -1).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_ties_and_grid(fmt):
    """Every grid value and every midpoint, times scales that make the quotients exact: ties to the even code."""

    from representax_b200.ops.fp4 import dequantize, quantize

    half = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=_dev())
    even = torch.tensor([0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0], device=_dev())
    grid = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6], device=_dev())
    size = 32 if fmt == "mxfp4" else 16
    for mult in ((1.0, 2.0 ** -20, 2.0 ** 30) if fmt == "mxfp4" else (1.0, 1.125, 1.875, 208.0)):
        x = torch.zeros(2, 2 * size, device=_dev())
        x[0, 0], x[0, 1:8] = 6.0, half
        x[0, size], x[0, size + 1:size + 8] = -6.0, -half
        x[1, :8], x[1, size:size + 8] = grid, -grid
        x *= mult
        if fmt == "nvfp4":  # a block of 448 * 6 puts the row factor at 1, so the scale of the others is `mult`
            x = torch.cat([x, torch.full((2, 16), 448.0 * 6, device=_dev())], 1)
        v = dequantize(quantize(x, fmt), torch.float32)
        assert torch.equal(v[0, 1:8], even * mult) and torch.equal(v[0, size + 1:size + 8], -even * mult)
        assert torch.equal(v[1, :8], grid * mult) and torch.equal(v[1, size:size + 8], -grid * mult)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_extremes(fmt, dtype):
    from representax_b200.ops.fp4 import dequantize, quantize

    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros(6, 96, dtype=dtype, device=_dev())
    x[1] = big
    x[2, ::2], x[2, 1::2] = tiny, -tiny / 4
    x[3, 40] = float("nan")
    x[4, 70] = float("-inf")
    x[5] = torch.linspace(-1, 1, 96)
    op = quantize(x, fmt)
    v = dequantize(op, torch.float32)
    ref = dequantize(quantize(x.cpu(), fmt), torch.float32)
    assert torch.equal(v.cpu().nan_to_num(nan=-7.0), ref.nan_to_num(nan=-7.0))
    assert bool((v[0] == 0).all()) and v[2].isfinite().all()
    # the nearest grid value of the widest types' largest number is 2^128, which fp32 does not hold
    assert bool((v[1] == (65536.0 if dtype == torch.float16 and fmt == "mxfp4" else v[1, 0])).all())
    assert v[1].isinf().all() if dtype != torch.float16 else v[1].isfinite().all()
    block = 32 if fmt == "mxfp4" else 96  # NVFP4: the row's factor is NaN
    assert v[3, 40 // block * block:][:block].isnan().all() and v[4, 70 // block * block:][:block].isnan().all()
    assert int(v.isnan().sum()) == 2 * block


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_strided_rows(fmt):
    from representax_b200.ops.fp4 import quantize

    wide = _randn(50, 300, seed=3)
    for view in (wide[:, 5:261], wide[::2, 8:264], wide.T[:200], wide[:1].expand(20, 300)):
        _same(quantize(view, fmt), quantize(view.contiguous().cpu(), fmt))
    empty = quantize(wide[:0], fmt)
    assert empty.rows == 0 and empty.k == 300


SIZES = [(1, 128, 256), (1, 300, 64), (1, 12288, 256), (7, 1, 32), (16, 128, 512), (17, 200, 96), (33, 33, 33), (64, 1000, 1000),
         (65, 129, 300), (128, 256, 256), (129, 3330, 40), (300, 520, 1000), (513, 2050, 384), (1000, 2048, 2048), (2000, 777, 1344),
         (40, 64, 20000), (100, 300, 2500), (300, 521, 2500), (129, 64, 4111)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(fmt, m, n, k):
    from representax_b200.ops.fp4 import dequantize, gemm, linear_fp4, quantize

    x, w = _randn(m, k, seed=m + k), _randn(n, k, seed=n, std=k ** -0.5)
    b = _randn(n, seed=1) if n % 2 else None
    res = _randn(m, n, seed=2) if m % 2 else None
    wq, xq = quantize(w, fmt), quantize(x, fmt)
    y = linear_fp4(x, wq, b, res)
    _status_ok()
    want = dequantize(xq, torch.float32).double() @ dequantize(wq, torch.float32).double().T
    want = want if b is None else want + b.double()
    want = want if res is None else want + res.double()
    assert y.dtype == torch.bfloat16 and _rel(y, want) < TOL
    assert torch.equal(gemm(xq, wq, bias=b, residual=res), y)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(16, 72, 64), (17, 72, 64), (32, 72, 700), (33, 72, 700), (33, 72, 800), (64, 300, 1100), (65, 300, 1700),
                                   (65, 300, 2000), (300, 1024, 2000), (300, 1100, 2000), (2000, 200, 2000)])
def test_linear_on_both_sides_of_the_few_row_bounds(fmt, m, n, k):
    from representax_b200.ops.fp4 import dequantize, linear_fp4, quantize

    x, w, res = _randn(m, k, seed=m + k), _randn(n, k, seed=n, std=k ** -0.5), _randn(m, n, seed=2)
    wq = quantize(w, fmt)
    y = linear_fp4(x, wq, None, res)
    _status_ok()
    want = dequantize(quantize(x, fmt), torch.float32).double() @ dequantize(wq, torch.float32).double().T + res.double()
    assert _rel(y, want) < TOL


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [3, 200])
def test_linear_of_parts_and_views(fmt, m):
    from representax_b200.ops.fp4 import linear_fp4, quantize

    w = _randn(2 * 200, 96, seed=1)
    x, b, res = _randn(m, 96, seed=2), _randn(400, seed=3), _randn(m, 400, seed=4)
    whole = linear_fp4(x, quantize(w, fmt), b, res)
    parts = quantize(w, fmt, parts=2)
    assert torch.equal(linear_fp4(x, parts, b, res), whole)
    one = parts.part(1)
    assert torch.equal(linear_fp4(x, one, b[200:].contiguous(), res[:, 200:]), whole[:, 200:])
    wide = torch.zeros(m, 99, dtype=torch.bfloat16, device=_dev())
    wide[:, 3:] = x
    assert torch.equal(linear_fp4(wide[:, 3:], parts, b, res.T.contiguous().T), whole)
    flat = torch.zeros(m * 400 + 1, dtype=torch.bfloat16, device=_dev())
    flat[1:] = res.reshape(-1)
    assert torch.equal(linear_fp4(x, parts, b, flat[1:].view(m, 400)), whole)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 5, 300])
def test_single_column_of_any_stride(fmt, m):
    """One output column, one contraction value: their strides mean nothing, whatever they are."""

    from representax_b200.ops.fp4 import gemm, linear_fp4, quantize

    x, w = _randn(m, 64, seed=1), quantize(_randn(1, 64, seed=2), fmt)
    res = _randn(7, m, seed=3)[2:3].T  # strides (1, m)
    want = linear_fp4(x, w, None, res.clone(memory_format=torch.contiguous_format))
    assert torch.equal(linear_fp4(x, w, None, res), want)
    assert torch.equal(gemm(quantize(x, fmt), w, residual=res), want)
    column, thin = _randn(3, m, seed=4)[1:2].T, quantize(_randn(40, 1, seed=5), fmt)
    assert torch.equal(linear_fp4(column, thin), linear_fp4(column.clone(memory_format=torch.contiguous_format), thin))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (70, 203, 301), (300, 512, 256)])
def test_linear_gradients(fmt, m, n, k):
    """dx = dy Q(W), the bias and residual gradients; one bf16 rounding each."""

    from representax_b200.ops.fp4 import dequantize, linear_fp4, quantize

    w = quantize(_randn(n, k, seed=1, std=k ** -0.5), fmt)
    x, b, res, dy = _randn(m, k, seed=2).requires_grad_(), _randn(n, seed=3).requires_grad_(), _randn(m, n, seed=4), _randn(m, n, seed=5)
    res.requires_grad_()
    dx, db, dres = torch.autograd.grad(linear_fp4(x, w, b, res), [x, b, res], dy)
    _status_ok()
    assert _rel(dx, dy.double() @ dequantize(w, torch.float32).double()) < TOL
    assert _rel(db, dy.double().sum(0)) < TOL and torch.equal(dres, dy)
    wide = torch.nn.Parameter(b.detach().float())  # an fp32 parameter: its gradient stays fp32
    dx2, db2 = torch.autograd.grad(linear_fp4(x, w, wide), [x, wide], dy)
    assert torch.equal(dx2, dx) and db2.dtype == torch.float32 and _rel(db2, dy.double().sum(0)) < 1e-5


def _act(g, name):
    from representax_b200.ops.nn import _act_reference

    return _act_reference(g, name)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t,h,i", [(1, 256, 128), (5, 96, 200), (16, 64, 40), (32, 512, 384), (33, 512, 384), (100, 256, 130), (300, 256, 1000),
                                   (513, 768, 1152)])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "quick_gelu"])
def test_feed_forward(fmt, t, h, i, act):
    """Against the formula with the hidden state quantised from 64 bits (NVFP4: from its bf16 rounding). Where a
    hidden value lies on a rounding boundary the last bit of fp32 decides, so a few codes may differ (a share below
    2^-13 of them, by one step of about a quarter: 2^-8.5 of the result at most)."""

    from representax_b200.ops.fp4 import dequantize, fake_quantize_reference, gated_feed_forward_fp4, quantize

    x, w1, w2 = _randn(t, h, seed=1), _randn(2 * i, h, seed=2, std=h ** -0.5), _randn(h, i, seed=3, std=i ** -0.5)
    b1, b2, res = _randn(2 * i, seed=4, std=0.2), _randn(h, seed=5), _randn(t, h, seed=6)
    q1, q2 = quantize(w1, fmt, parts=2), quantize(w2, fmt)
    y = gated_feed_forward_fp4(x, q1, q2, activation=act, gate_up_bias=b1, down_bias=b2, residual=res)
    _status_ok()
    z = fake_quantize_reference(x, fmt).double() @ dequantize(q1, torch.float32).double().T + b1.double()
    hidden = _act(z[:, :i], act) * z[:, i:]
    hidden = hidden.float() if fmt == "mxfp4" else hidden.to(torch.bfloat16)
    want = fake_quantize_reference(hidden, fmt).double() @ dequantize(q2, torch.float32).double().T + b2.double() + res.double()
    assert _rel(y, want) < TOL + 2.0 ** -8.5


@pytest.mark.parametrize("fmt", FMTS)
def test_feed_forward_under_grad(fmt):
    """With gradients the block runs as separate layers: the input gradient of those layers."""

    from representax_b200.ops.fp4 import dequantize, gated_feed_forward_fp4, linear_fp4, quantize
    from representax_b200.ops.nn import gated_activation

    x, dy = _randn(70, 64, seed=1).requires_grad_(), _randn(70, 64, seed=7)
    q1, q2 = quantize(_randn(192, 64, seed=2, std=0.125), fmt, parts=2), quantize(_randn(64, 96, seed=3, std=0.1), fmt)
    (dx,) = torch.autograd.grad(gated_feed_forward_fp4(x, q1, q2, activation="silu"), [x], dy)
    z = linear_fp4(x.detach(), q1).double().requires_grad_()
    (dz,) = torch.autograd.grad(_act(z[:, :96], "silu") * z[:, 96:], [z], dy.double() @ dequantize(q2, torch.float32).double())
    # dh, dz and dx are each rounded to bf16
    assert _rel(dx, dz @ dequantize(q1, torch.float32).double()) < 3 * 2.0 ** -9
    assert gated_activation(linear_fp4(x.detach(), q1), "silu").shape == (70, 96)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t,h,i", [(1, 64, 40), (20, 96, 200), (70, 256, 130), (300, 256, 384)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_feed_forward_value_and_gradients(fmt, t, h, i, act):
    """The value is the same with and without gradients. Gradients against those of the separate layers in 64 bits (dh, dz
    and dx, or the bias gradient, are each rounded to bf16, at most 2^-9 each)."""

    from representax_b200.ops.fp4 import dequantize, gated_feed_forward_fp4, linear_fp4, quantize

    q1, q2 = quantize(_randn(2 * i, h, seed=2, std=h ** -0.5), fmt, parts=2), quantize(_randn(h, i, seed=3, std=i ** -0.5), fmt)
    x, dy = _randn(t, h, seed=1), _randn(t, h, seed=7)
    b1, b2, res = _randn(2 * i, seed=4, std=0.2), _randn(h, seed=5), _randn(t, h, seed=6)
    run = lambda x, b1, b2, res: gated_feed_forward_fp4(x, q1, q2, activation=act, gate_up_bias=b1, down_bias=b2, residual=res)  # noqa: E731
    want = run(x, b1, b2, res)
    leaves = [v.clone().requires_grad_() for v in (x, b1, b2, res)]
    y = run(*leaves)
    assert torch.equal(y.detach(), want)
    dx, db1, db2, dres = torch.autograd.grad(y, leaves, dy)
    _status_ok()
    z = linear_fp4(x, q1, b1).double().requires_grad_()
    (dz,) = torch.autograd.grad(_act(z[:, :i], act) * z[:, i:], [z], dy.double() @ dequantize(q2, torch.float32).double())
    assert _rel(dx, dz @ dequantize(q1, torch.float32).double()) < 3 * 2.0 ** -9
    assert _rel(db1, dz.sum(0)) < 3 * 2.0 ** -9 and _rel(db2, dy.double().sum(0)) < TOL and torch.equal(dres, dy)
    for k, leaf in enumerate(leaves):  # one gradient at a time
        args = [v if j != k else leaf for j, v in enumerate((x, b1, b2, res))]
        (g,) = torch.autograd.grad(run(*args), [leaf], dy)
        assert _rel(g, (dx, db1, db2, dres)[k].double()) < 2.0 ** -8
    wide = torch.nn.Parameter(b1.float())  # an fp32 parameter with an accumulator
    wide.main_grad = torch.ones_like(wide.data)
    run(x, wide, b2, res).backward(dy)
    assert wide.grad is None and _rel(wide.main_grad - 1, dz.sum(0)) < 3 * 2.0 ** -9
    none = run(x[:0].clone().requires_grad_(), b1, b2, res[:0])
    assert none.shape == (0, h)


@pytest.mark.parametrize("fmt", FMTS)
def test_feed_forward_gradient_of_no_rows(fmt):
    from representax_b200.ops.fp4 import gated_feed_forward_fp4, quantize

    q1, q2 = quantize(_randn(96, 64, seed=2), fmt, parts=2), quantize(_randn(64, 48, seed=3), fmt)
    x, b = _randn(0, 64).requires_grad_(), _randn(96, seed=4).requires_grad_()
    dx, db = torch.autograd.grad(gated_feed_forward_fp4(x, q1, q2, activation="silu", gate_up_bias=b), [x, b], _randn(0, 64))
    assert dx.shape == (0, 64) and bool((db == 0).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [5, 300])
def test_nonfinite_rows_stay_rows(fmt, m):
    from representax_b200.ops.fp4 import gated_feed_forward_fp4, linear_fp4, quantize

    x, w = _randn(m, 128, seed=1), quantize(_randn(64, 128, seed=2), fmt)
    bad = x.clone()
    bad[1, 7], bad[3, 100] = float("nan"), float("inf")
    keep = [r for r in range(m) if r not in (1, 3)]
    y, clean = linear_fp4(bad, w), linear_fp4(x, w)
    assert torch.equal(y[keep], clean[keep]) and y[1].isnan().all() and y[3].isnan().all()
    w1, w2 = quantize(_randn(192, 128, seed=3, std=0.1), fmt, parts=2), quantize(_randn(128, 96, seed=4, std=0.1), fmt)
    y, clean = (gated_feed_forward_fp4(v, w1, w2, activation="silu") for v in (bad, x))
    assert torch.equal(y[keep], clean[keep]) and y[1].isnan().all() and y[3].isnan().all()
    assert torch.equal(linear_fp4(x[:0], w), x.new_empty(0, 64))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 100, 700])
def test_other_stream_and_repeats(fmt, m):
    from representax_b200.ops.fp4 import gated_feed_forward_fp4, quantize

    x = _randn(m, 512, seed=1)
    w1, w2 = quantize(_randn(2 * 384, 512, seed=2, std=0.04), fmt, parts=2), quantize(_randn(512, 384, seed=3, std=0.05), fmt)
    run = lambda: gated_feed_forward_fp4(x, w1, w2, activation="silu", residual=x)  # noqa: E731
    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [run() for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(first, a) for a in again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    graph.replay()
    _status_ok()
    assert torch.equal(y, first)


def test_refusals():
    from representax_b200.ops import fp4 as F
    from representax_b200.ops._ext import ext, status

    x = _randn(4, 64)
    w = F.quantize(_randn(32, 64), "nvfp4")
    with pytest.raises(ValueError, match="fmt"):
        F.quantize(x, "fp4")
    with pytest.raises(TypeError, match="bfloat16"):
        F.quantize(x.double())
    with pytest.raises(ValueError, match="parts"):
        F.quantize(x, parts=3)
    with pytest.raises(ValueError, match="column"):
        F.quantize(x[:, :0])
    with pytest.raises(ValueError, match="contract"):
        F.linear_fp4(x[:, :32], w)
    with pytest.raises(ValueError, match="bias"):
        F.linear_fp4(x, w, x[0])
    with pytest.raises(ValueError, match="residual"):
        F.linear_fp4(x, w, None, x)
    with pytest.raises(TypeError, match="residual"):
        F.linear_fp4(x, w, None, torch.zeros(4, 32, device=_dev()))
    with pytest.raises(ValueError, match="is on"):
        F.linear_fp4(x.cpu(), w)
    with pytest.raises(ValueError, match="one format"):
        F.gemm(F.quantize(x, "mxfp4"), w)
    with pytest.raises(ValueError, match="parts=2"):
        F.gated_feed_forward_fp4(x, w, w, activation="silu")
    with pytest.raises(ValueError, match="activation"):
        F.gated_feed_forward_fp4(x, w, w, activation="relu6")
    with pytest.raises(RuntimeError, match="scales must be"):  # an operand whose scales are cut short
        ext().fp4_linear(x, w.data, w.scales[:, :2], w.row_scale, 1, 2, None, None, status(_dev()))
    with pytest.raises(RuntimeError, match="rows of codes"):
        ext().fp4_linear(x, w.data[:, :16], w.scales, w.row_scale, 1, 2, None, None, status(_dev()))


@pytest.mark.parametrize("fmt", FMTS)
def test_model_with_4bit_weights(fmt):
    """A small Qwen3 tower: every layer's linear runs 4-bit products. Against the same tower whose weights hold the
    dequantised values and whose activations stay bf16, one layer differs by the activations' quantisation, whose
    relative error is at most 1/6 (half a step between 4 and 6) and about 1/10 in the mean square; three
    products in a row on the residual branch stay below 1/2."""

    from representax_b200.models import FP4Weight, quantize_linears_fp4
    from representax_b200.models.qwen3 import Qwen3TextConfig, Qwen3TextTower
    from representax_b200.ops import nn as N

    cfg = Qwen3TextConfig(vocab_size=100, hidden_size=128, intermediate_size=264, num_hidden_layers=1, num_attention_heads=2,
                          num_key_value_heads=2, head_dimension=64)
    tower = Qwen3TextTower(cfg, torch.Generator().manual_seed(0)).to(_dev())
    plain = Qwen3TextTower(cfg, torch.Generator().manual_seed(0)).to(_dev())
    quantize_linears_fp4(tower, fmt=fmt)
    layer, other = tower.layers[0], plain.layers[0]
    assert isinstance(layer.gate_up, FP4Weight) and layer.gate_up.parts == 2 and not tower.embed_tokens.requires_grad
    with torch.no_grad():
        for name in ("qkv", "o_proj", "gate_up", "down"):
            getattr(other, name).copy_(getattr(layer, name).dequantized())
    seg = N.Segments.from_lengths([40, 3], _dev())
    emb = torch.randn(seg.total, 128, device=_dev()).to(torch.bfloat16)
    pos = torch.cat([torch.arange(n) for n in seg.lengths()]).to(_dev())
    with torch.no_grad():
        a, b = tower(emb, seg, pos), plain(emb, seg, pos)
    _status_ok()
    assert a.isfinite().all() and not torch.equal(a, b) and _rel(a, b) < 0.5
    state = tower.state_dict()
    again = quantize_linears_fp4(Qwen3TextTower(cfg, torch.Generator().manual_seed(1)).to(_dev()), fmt=fmt)
    again.load_state_dict(state)
    with torch.no_grad():
        assert torch.equal(again(emb, seg, pos), a)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("c", [1, 9, 511, 1029, 2600])
def test_quantize_rows_at_any_address(fmt, dtype, c):
    from representax_b200.ops.fp4 import quantize

    flat = _randn(4 * (c + 9) + 16, seed=c, dtype=dtype)
    for offset in range(9):
        for pitch in (c, c + 9):
            x = flat[offset:offset + 3 * pitch + c].as_strided((4, c), (pitch, 1))
            _same(quantize(x, fmt), quantize(x.contiguous().cpu(), fmt))
