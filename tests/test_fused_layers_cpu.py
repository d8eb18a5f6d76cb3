"""Where a model's gated feed-forward block goes, without a GPU."""

import pytest
import torch

from representax_b200.ops import ffn
from representax_b200.ops import nn as N


@pytest.mark.parametrize("hidden,width", [(16, 10), (10, 16), (12, 20)])
def test_widths_that_the_kernels_do_not_take_keep_the_separate_layers(hidden, width, monkeypatch):
    g = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    args = (n(5, hidden), n(2 * width, hidden), n(hidden, width), "silu", n(2 * width), n(hidden))
    x = args[0]
    want = N.gated_mlp(*args, residual=x)
    monkeypatch.setattr(N, "native", lambda t: t is x)  # (the separate layers are plain products at these widths)
    monkeypatch.setattr(ffn, "gated_feed_forward", lambda *a, **k: pytest.fail("the block's kernels do not take these widths"))
    with N.fused_feed_forward():
        assert torch.equal(N.gated_mlp(*args, residual=x), want)

