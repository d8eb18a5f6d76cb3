"""Launches of the feed-forward block and of the 4-bit layers, forward and backward."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(*shape):
    return torch.randn(*shape, device="cuda").to(torch.bfloat16)


def _count(fn):
    from representax_b200.ops._ext import launch_counter

    counter = launch_counter()
    counter.launches, counter.counting = 0, True
    try:
        fn()
    finally:
        counter.counting = False
    return counter.launches


@pytest.mark.parametrize("t", [1, 20, 300])
@pytest.mark.parametrize("bias", [False, True])
def test_feed_forward(t, bias):
    from representax_b200.ops.ffn import gated_feed_forward

    x, w1, w2, dy = _randn(t, 64), _randn(192, 64), _randn(64, 96), _randn(t, 64)
    b1, b2 = (_randn(192), _randn(64)) if bias else (None, None)
    run = lambda: gated_feed_forward(x, w1, w2, activation="silu", gate_up_bias=b1, down_bias=b2)  # noqa: E731
    assert _count(run) == 2
    leaves = [v.requires_grad_() for v in (x, w1, w2, b1, b2) if v is not None]
    # forward 2; ddown, dz, dgate_up, dx; the two bias gradients
    assert _count(lambda: torch.autograd.grad(run(), leaves, dy)) == 6 + 2 * bias
    store = [torch.nn.Parameter(v.detach().float()) for v in (w1, w2)]  # the Python node's parameters
    for p in store:
        p.main_grad = torch.zeros_like(p.data)
    assert _count(lambda: gated_feed_forward(x, *store, activation="silu").backward(dy)) == 6
    only = w2.detach().requires_grad_()
    x0, w10 = x.detach(), w1.detach()
    assert _count(lambda: gated_feed_forward(x0, w10, only, activation="silu").backward(dy)) == 3


@pytest.mark.parametrize("fmt,block", [("mxfp4", 3), ("nvfp4", 4)])
@pytest.mark.parametrize("t", [1, 300])
def test_4bit_layers(fmt, block, t):
    from representax_b200.ops import fp4 as F

    x, dy, b = _randn(t, 64), _randn(t, 64), _randn(64)
    w1, w2 = F.quantize(_randn(192, 64), fmt, parts=2), F.quantize(_randn(64, 96), fmt)
    w = F.quantize(_randn(64, 64), fmt)
    assert _count(lambda: F.quantize(x, fmt)) == 1 and _count(lambda: F.dequantize(w)) == 1
    assert _count(lambda: F.linear_fp4(x, w, b)) == 2 and _count(lambda: F.linear_fp4(x, w1)) == 3
    xq = F.quantize(x, fmt)
    assert _count(lambda: F.gemm(xq, w)) == 1
    assert _count(lambda: F.gated_feed_forward_fp4(x, w1, w2, activation="silu")) == block
    assert _count(lambda: F.linear_fp4(x[:0], w)) == 0
    xg, bg = x.clone().requires_grad_(), b.clone().requires_grad_()
    # forward 2, decoder and product of dx, bias gradient
    assert _count(lambda: torch.autograd.grad(F.linear_fp4(xg, w, bg), [xg, bg], dy)) == 5
