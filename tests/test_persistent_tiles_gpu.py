"""Products whose CTA pairs work through several tiles each: more than twice and more than three times the 74 pairs of
the GPU. What one tile never shows is then on the path: an accumulator used again, scales and stages carried
over a tile's end, the next tile's residual. Ragged in every dimension, against 64 bits.

Tolerances (2-norm of the difference over that of the result): a rounding to bf16 is below 2^-9 in the 2-norm (half a step is
at most 2^-8 of a value and a third of its square on average), fp32 accumulation below 2^-12. The block rounds h (or dz) and
y (or the gradient) and keeps 11 bits: 2^-8 in all. Codes of h that lie on a rounding boundary may differ as the last bit
of fp32 decides: a share below 2^-13, by a quarter at most, 2^-8.5 of the result.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

FMTS = ("mxfp4", "nvfp4")
TOL = 2.0 ** -9 + 2.0 ** -12


def _dev():
    return torch.device("cuda", 0)


def _status_ok():
    from representax_b200.ops._ext import check_status

    torch.cuda.synchronize()
    check_status(_dev())


def _rel(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm())


def _worst_tile(got, want):
    """The largest relative difference of any 256 x 256 tile: a wrong tile does not drown in the right ones."""

    rows, cols = got.shape
    worst = 0.0
    for r in range(0, rows, 256):
        for c in range(0, cols, 256):
            worst = max(worst, _rel(got[r:r + 256, c:c + 256], want[r:r + 256, c:c + 256]))
    return worst


def _randn(*shape, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=_dev()) * std).to(torch.bfloat16)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [4100, 4104])  # rows of any address, and 16-byte aligned ones
@pytest.mark.parametrize("k", [40, 300, 1300, 1536 + 64])  # 1, 2, 6 and 7 stages: the ring of five ends elsewhere in every tile
def test_4bit_product(fmt, n, k):
    from representax_b200.ops.fp4 import dequantize, linear_fp4, quantize

    m = 4097  # 17 x 17 tiles: 289
    x, w, b, res = _randn(m, k, seed=1), _randn(n, k, seed=2, std=k ** -0.5), _randn(n, seed=3), _randn(m, n, seed=4)
    wq = quantize(w, fmt)
    want = dequantize(quantize(x, fmt), torch.float32).double() @ dequantize(wq, torch.float32).double().T + b.double() + res.double()
    y = linear_fp4(x, wq, b, res)
    _status_ok()
    assert _rel(y, want) < TOL and _worst_tile(y, want) < 1.5 * TOL
    plain = linear_fp4(x, wq)
    _status_ok()
    assert _rel(plain, want - b.double() - res.double()) < TOL


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t,i", [(2049, 2312), (2049, 3336), (4100, 3330)])  # 171, 243 and 459 gated tiles
def test_4bit_block(fmt, t, i):
    from representax_b200.ops.fp4 import dequantize, fake_quantize_reference, gated_feed_forward_fp4, quantize

    h = 300
    x, w1, w2 = _randn(t, h, seed=1), _randn(2 * i, h, seed=2, std=h ** -0.5), _randn(h, i, seed=3, std=i ** -0.5)
    b1, res = _randn(2 * i, seed=4, std=0.2), _randn(t, h, seed=5)
    q1, q2 = quantize(w1, fmt, parts=2), quantize(w2, fmt)
    y = gated_feed_forward_fp4(x, q1, q2, activation="silu", gate_up_bias=b1, residual=res)
    _status_ok()
    z = fake_quantize_reference(x, fmt).double() @ dequantize(q1, torch.float32).double().T + b1.double()
    hidden = torch.nn.functional.silu(z[:, :i]) * z[:, i:]
    hidden = hidden.float() if fmt == "mxfp4" else hidden.to(torch.bfloat16)
    want = fake_quantize_reference(hidden, fmt).double() @ dequantize(q2, torch.float32).double().T + res.double()
    assert _rel(y, want) < TOL + 2.0 ** -8.5
    assert max(_rel(y[r:r + 128], want[r:r + 128]) for r in range(0, t, 128)) < 2 * (TOL + 2.0 ** -8.5)


@pytest.mark.parametrize("t,i", [(4100, 2312), (4100, 3400)])  # 323 and 459 gated tiles, 170 and 238 of dz
@pytest.mark.parametrize("bias", [False, True])
def test_block_forward_and_gradients(t, i, bias):
    from representax_b200.ops.ffn import gated_feed_forward

    h = 72
    o = {"x": _randn(t, h, seed=1), "w1": _randn(2 * i, h, seed=2, std=h ** -0.5), "w2": _randn(h, i, seed=3, std=i ** -0.5),
         "res": _randn(t, h, seed=4)}
    if bias:
        o["b1"], o["b2"] = _randn(2 * i, seed=5, std=0.2), _randn(h, seed=6, std=0.2)
    dy = _randn(t, h, seed=7)

    def formula(v):
        z = v["x"] @ v["w1"].T + (v["b1"] if bias else 0)
        y = (torch.nn.functional.silu(z[:, :i]) * z[:, i:]) @ v["w2"].T + (v["b2"] if bias else 0)
        return y + v["res"]

    run = lambda v: gated_feed_forward(v["x"], v["w1"], v["w2"], activation="silu", gate_up_bias=v.get("b1"),  # noqa: E731
                                       down_bias=v.get("b2"), residual=v["res"])
    ref = {k: v.double().requires_grad_() for k, v in o.items()}
    want_y = formula(ref)
    want = torch.autograd.grad(want_y, list(ref.values()), dy.double())
    want_y = want_y.detach()
    y = run(o)
    _status_ok()
    rows = lambda a, b: max(_rel(a[r:r + 128], b[r:r + 128]) for r in range(0, len(b), 128))  # noqa: E731
    assert _rel(y, want_y) < 2.0 ** -8 and rows(y, want_y) < 2.0 ** -7
    leaves = {k: v.clone().requires_grad_() for k, v in o.items()}
    y = run(leaves)
    assert _rel(y.detach(), want_y) < 2.0 ** -8 and rows(y.detach(), want_y) < 2.0 ** -7
    got = torch.autograd.grad(y, list(leaves.values()), dy)
    _status_ok()
    for name, a, b in zip(o, got, want):
        assert _rel(a, b) < 2.0 ** -8, name
        if a.dim() == 2:
            assert rows(a, b) < 2.0 ** -7, name
