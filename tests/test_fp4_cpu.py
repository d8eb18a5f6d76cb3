"""Microscaled 4-bit formats and the gated feed-forward block on the CPU: the
PyTorch statements, the storage layout, dispatch and refusals."""

import pytest
import torch

from representax_b200.ops import fp4 as F
from representax_b200.ops import nn as N
from representax_b200.ops.ffn import gated_feed_forward

FMTS = ("mxfp4", "nvfp4")


def _loop_quantize(x, fmt):
    """The definition, value by value."""

    import math

    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    size = F.BLOCK[fmt]
    out = torch.zeros_like(x, dtype=torch.float64)

    def nearest(v):
        best = min(range(8), key=lambda c: (abs(abs(v) - grid[c]), c % 2))
        return math.copysign(grid[best], v)

    for r in range(x.shape[0]):
        row = [float(v) for v in x[r]]
        top = max(abs(v) for v in row)
        factor = 2.0 ** math.ceil(math.log2(top / 2688)) if top else 1.0
        for c0 in range(0, len(row), size):
            block = row[c0:c0 + size]
            amax = max(abs(v) for v in block)
            if fmt == "mxfp4":
                scale = 2.0 ** math.ceil(math.log2(amax / 6)) if amax else 1.0
            else:
                scale = float(torch.tensor(amax / 6 / factor).to(torch.float8_e4m3fn).float()) * factor
            for i, v in enumerate(block):
                out[r, c0 + i] = nearest(v / scale) * scale if scale else 0.0
    return out


@pytest.mark.parametrize("fmt", FMTS)
def test_statement_is_the_definition(fmt):
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(6, 70, generator=g) * torch.logspace(-2, 2, 6)[:, None]).to(torch.bfloat16)
    x[3, 32:64] = 0
    assert torch.equal(F.fake_quantize_reference(x, fmt).double(), _loop_quantize(x, fmt))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,k,parts", [(1, 1, 1), (5, 33, 1), (260, 300, 2), (128, 256, 1)])
def test_layout(fmt, rows, k, parts):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, k, generator=g)
    op = F.quantize(x, fmt, parts=parts)
    assert op.shape == (rows, k) and op.data.shape == (rows, (k + 31) // 32 * 16)
    values = F.fake_quantize_reference(x, fmt)
    assert torch.equal(F.dequantize(op, torch.float32), values)
    # the scale of (row, block) by its stated position
    size, per = F.BLOCK[fmt], rows // parts
    tiles, groups = (per + 127) // 128, op.scales.shape[1]
    flat = op.scales.reshape(-1)
    scales = F.scale_values(op)
    for r in range(0, rows, 37):
        part, q = divmod(r, per)
        for b in range(-(-k // size)):
            at = ((part * tiles + q // 128) * groups + b // 4) * 512 + 16 * (q % 32) + 4 * (q % 128 // 32) + b % 4
            byte = flat[at]
            want = 2.0 ** (int(byte) - 127) if fmt == "mxfp4" else float(byte.view(torch.float8_e4m3fn).float())
            assert float(scales[r, b]) == want
    for i in range(parts):
        cut = slice(i * per, (i + 1) * per)
        assert torch.equal(F.dequantize(op.part(i), torch.float32), values[cut])


@pytest.mark.parametrize("fmt", FMTS)
def test_values_are_fixed_points_and_near(fmt):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20, 128, generator=g)
    v = F.fake_quantize_reference(x, fmt)
    assert torch.equal(F.fake_quantize_reference(v, fmt), v) or fmt == "nvfp4"
    # half a step of the top of the grid is 1/6 of the block's largest scaled value; an E4M3 scale is off by 2^-4
    top = x.abs().reshape(20, -1, F.BLOCK[fmt]).amax(-1).repeat_interleave(F.BLOCK[fmt], 1)
    bound = top * (1 / 6 * 2 if fmt == "mxfp4" else 1 / 6 * (1 + 2 ** -4) + 2 ** -4)
    assert bool(((x - v).abs() <= bound).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_statement_and_gradients(fmt):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(7, 40, generator=g, requires_grad=True)
    w = F.quantize(torch.randn(12, 40, generator=g), fmt)
    b = torch.randn(12, generator=g, requires_grad=True)
    res = torch.randn(7, 12, generator=g, requires_grad=True)
    y = F.linear_fp4(x, w, b, res)
    wv = F.dequantize(w, torch.float32)
    want = F.fake_quantize_reference(x.detach(), fmt) @ wv.T + b + res
    torch.testing.assert_close(y, want, rtol=1e-5, atol=1e-5)
    dy = torch.randn(7, 12, generator=g)
    dx, db, dr = torch.autograd.grad(y, [x, b, res], dy)
    torch.testing.assert_close(dx, dy @ wv, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(db, dy.sum(0))
    assert torch.equal(dr, dy)


def test_feed_forward_statement():
    g = torch.Generator().manual_seed(3)
    x, w1, w2 = torch.randn(5, 12, generator=g), torch.randn(28, 12, generator=g), torch.randn(12, 14, generator=g)
    for act in ("silu", "gelu", "gelu_tanh", "quick_gelu"):
        y = gated_feed_forward(x, w1, w2, activation=act, residual=x)
        z = x @ w1.T
        torch.testing.assert_close(y, (N._act_reference(z[:, :14], act) * z[:, 14:]) @ w2.T + x)
    with pytest.raises(ValueError, match="gate_up must be"):
        gated_feed_forward(x, w1[:26], w2, activation="silu")
    with pytest.raises(ValueError, match="activation"):
        gated_feed_forward(x, w1, w2, activation="tanh")


@pytest.mark.parametrize("fmts", [("mxfp4", "mxfp4"), ("nvfp4", "nvfp4"), ("mxfp4", "nvfp4")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_feed_forward_rounds_where_the_kernels_round(fmts, dtype):
    """h is quantised from fp32 in MXFP4 and from the rows' type where NVFP4 is involved; y is rounded once. With and
    without gradients."""

    g = torch.Generator().manual_seed(8)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    x, b1, b2, res = n(30, 64), n(96), n(64), n(30, 64)
    q1, q2 = F.quantize(n(96, 64) / 8, fmts[0], parts=2), F.quantize(n(64, 48) / 7, fmts[1])
    z = F.fake_quantize_reference(x, fmts[0]) @ F.dequantize(q1, torch.float32).T + b1.float()
    h = N._act_reference(z[:, :48], "silu") * z[:, 48:]
    h = h if fmts == ("mxfp4", "mxfp4") else h.to(dtype).float()
    want = (F.fake_quantize_reference(h, fmts[1]) @ F.dequantize(q2, torch.float32).T + b2.float() + res.float()).to(dtype)
    run = lambda x: F.gated_feed_forward_fp4(x, q1, q2, activation="silu", gate_up_bias=b1, down_bias=b2, residual=res)  # noqa: E731
    assert torch.equal(run(x), want)
    y = run(x.clone().requires_grad_())
    assert y.requires_grad and torch.equal(y.detach(), want)


def test_gated_mlp_keeps_the_separate_layers():
    """Models run the separate layers unless they are asked otherwise: the same bits as before."""

    g = torch.Generator().manual_seed(4)
    x, w1, w2 = torch.randn(5, 16, generator=g), torch.randn(48, 16, generator=g), torch.randn(16, 24, generator=g)
    b1, b2 = torch.randn(48, generator=g), torch.randn(16, generator=g)
    want = N.linear(N.gated_activation(N.linear(x, w1, b1), "silu"), w2, b2, residual=x)
    assert torch.equal(N.gated_mlp(x, w1, w2, "silu", b1, b2, residual=x), want)
    with N.fused_feed_forward():  # CPU rows: still the separate layers
        assert torch.equal(N.gated_mlp(x, w1, w2, "silu", b1, b2, residual=x), want)


@pytest.mark.parametrize("fmt", FMTS)
def test_weights_swapped_in_a_model(fmt):
    from representax_b200.models import FP4Weight, quantize_linears_fp4
    from representax_b200.models.modernvbert.config import ModernVBERTTextConfig
    from representax_b200.models.modernvbert.model import ModernBertTextTower

    cfg = ModernVBERTTextConfig(vocab_size=50, hidden_size=64, intermediate_size=40, num_hidden_layers=2, num_attention_heads=1)
    tower = ModernBertTextTower(cfg, torch.Generator().manual_seed(0))
    emb = torch.randn(9, 64, generator=torch.Generator().manual_seed(1))
    seg = N.Segments.from_lengths([4, 5], "cpu")
    pos = torch.cat([torch.arange(4), torch.arange(5)])
    before = tower(emb, seg, pos).detach()
    quantize_linears_fp4(tower, fmt=fmt, target_pattern=r"Wi|mlp_Wo")
    layer = tower.layers[0]
    assert isinstance(layer.Wi, FP4Weight) and layer.Wi.parts == 2 and layer.Wi.shape == (80, 64)
    assert isinstance(layer.Wqkv, torch.nn.Parameter) and not any(p.requires_grad for p in tower.parameters())
    after = tower(emb, seg, pos)
    assert after.isfinite().all() and not torch.equal(after, before)
    tower.to(torch.bfloat16)  # codes stay bytes, row factors fp32
    assert layer.Wi.data.dtype == torch.uint8 and (layer.Wi.row_scale is None or layer.Wi.row_scale.dtype == torch.float32)
    with pytest.raises(ValueError, match="target_pattern"):
        quantize_linears_fp4(ModernBertTextTower(cfg, torch.Generator().manual_seed(0)), target_pattern="nothing")
    with pytest.raises(ValueError, match="fmt"):
        FP4Weight(torch.zeros(4, 32), fmt="int4")


def test_feed_forward_refuses_weights_of_another_device():
    import copy

    x, q1, q2 = torch.randn(4, 64), F.quantize(torch.randn(96, 64), parts=2), F.quantize(torch.randn(64, 48))
    for first, second in ((True, False), (False, True), (True, True)):
        ops = []
        for op, away in ((q1, first), (q2, second)):
            op = copy.copy(op)
            if away:
                op.data, op.scales, op.row_scale = (t.to("meta") for t in (op.data, op.scales, op.row_scale))
            ops.append(op)
        with pytest.raises(ValueError, match="weights on"):
            F.gated_feed_forward_fp4(x, *ops, activation="silu")


def test_dequantize_refuses_an_output_of_another_shape():
    op = F.quantize(torch.randn(4, 40))
    for shape in ((4, 50), (4, 39), (5, 40), (160,), (1, 40), (2, 4, 40)):  # (50 columns take as many bytes of codes as 40)
        with pytest.raises(ValueError, match="out must be"):
            F.dequantize(op, out=torch.empty(shape))


def test_part_refuses_an_index_out_of_range():
    op = F.quantize(torch.randn(4, 40), parts=2)
    for index in (-1, 2):
        with pytest.raises(IndexError, match="of 2"):
            op.part(index)
    assert op.part(1).rows == 2


def test_refusals():
    x = torch.randn(4, 64)
    w = F.quantize(torch.randn(32, 64))
    for call, match in ((lambda: F.quantize(x, "e2m1"), "fmt"), (lambda: F.quantize(x[0]), "matrix"),
                        (lambda: F.quantize(x, parts=3), "parts"), (lambda: F.linear_fp4(x[:, :63], w), "contract"),
                        (lambda: F.linear_fp4(x, w, torch.zeros(3)), "bias"), (lambda: F.gemm(w, w, residual=x), "residual"),
                        (lambda: F.gemm(F.quantize(x, "mxfp4"), w), "one format"),
                        (lambda: F.gated_feed_forward_fp4(x, w, w, activation="silu"), "parts=2")):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(TypeError, match="float32"):
        F.quantize(x.double())
