"""Gated feed-forward block of the decoder and encoder layers.

``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual`` on packed
token rows, with the gate and up projections in one weight ``[Wg; Wu]``.

bf16 CUDA rows run hand-written kernels: one launch computes both
projections, the activation and the product (``csrc/gated.cu``; up to 32 rows, or
64 of narrow blocks, the weight-streaming kernel of ``csrc/few_rows.cu``), a second
one the down projection with bias and residual. The gate and up projections
are never written. For the backward pass the first launch also keeps
``act(g)`` and ``u act'(g)`` in 16 bits; the gradient of the block then takes
one launch for ``dz = [dh u act'(g) | dh act(g)]`` with ``dh = dy Wd`` (``dh`` is
never written) and the plain GEMMs for ``dx`` and the weights.

Anything else runs the PyTorch statement of the same formula.

Parity: the gated MLP blocks of src/representax/models/qwen3_vl/text.py and
src/representax/models/modernvbert/model.py.
"""

from __future__ import annotations

import torch

from ._ext import ext, status
from .functional import compute_view
from .nn import ACT_CODES as _CODES
from .nn import _act_reference


def _check(x, gate_up, down, activation, gate_up_bias, down_bias, residual) -> None:
    if activation not in _CODES:
        raise ValueError(f"unsupported activation {activation!r}")
    if x.dim() != 2 or gate_up.dim() != 2 or down.dim() != 2:
        raise ValueError("x, gate_up and down must be matrices")
    hidden, width = down.shape
    if x.shape[1] != hidden or gate_up.shape != (2 * width, hidden):
        raise ValueError(f"gate_up must be [2 I, H] and down [H, I] for x [T, H]: got {tuple(gate_up.shape)}, "
                         f"{tuple(down.shape)} and {tuple(x.shape)}")
    if gate_up_bias is not None and gate_up_bias.shape != (2 * width,):
        raise ValueError(f"gate_up_bias must be [{2 * width}]")
    if down_bias is not None and down_bias.shape != (hidden,):
        raise ValueError(f"down_bias must be [{hidden}]")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have the shape and type of x")


def wants_grad(*tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def plain(param) -> bool:
    """A bf16 tensor with nothing attached (compute copy, fp32 accumulator, shards): its own compute copy."""

    return param is None or (param.dtype is torch.bfloat16 and not param.__dict__)


def view(param):
    """The bf16 compute copy of a parameter, or None."""

    return param if plain(param) else compute_view(param)


def kernel_widths(hidden: int, width: int) -> bool:
    """Whether the kernels take blocks of these sizes (rows that the tensor maps can read: multiples of 16 bytes)."""

    return hidden % 8 == 0 and width % 8 == 0


class GatedFeedForwardFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_up, down, gate_up_bias, down_bias, residual, act):
        need = ctx.needs_input_grad
        through_z = need[0] or need[1] or need[3]
        y, h, saved, exps = ext().gated_ffn_forward(x, view(gate_up), view(down), view(gate_up_bias), view(down_bias),
                                                    residual, act, through_z, status(x.device))
        # kept only as far as the gradients asked for need it
        ctx.save_for_backward(x if need[1] else None, gate_up, down, gate_up_bias, down_bias, h if need[2] else None, saved,
                              exps)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gate_up, down, b1, b2, h, saved, exps = ctx.saved_tensors
        need = list(ctx.needs_input_grad[:5])
        params = (None, gate_up, down, b1, b2)
        acc = [None if p is None else getattr(p, "main_grad", None) for p in params]
        like = [dy.dtype if p is None else p.dtype for p in params]
        grads = ext().gated_ffn_backward(dy, x, h, view(gate_up), view(down), saved, exps, need, acc, like,
                                         status(dy.device))
        return (*grads, dy if ctx.needs_input_grad[5] else None, None)


def gated_feed_forward_reference(x, gate_up, down, activation, gate_up_bias=None, down_bias=None, residual=None):
    """The block in fp32, rounded once to the type of ``x``."""

    f = lambda t: None if t is None else t.float()  # noqa: E731
    z = torch.nn.functional.linear(x.float(), gate_up.float(), f(gate_up_bias))
    width = down.shape[1]
    y = torch.nn.functional.linear(_act_reference(z[:, :width], activation) * z[:, width:], down.float(), f(down_bias))
    return (y if residual is None else y + residual.float()).to(x.dtype)


def gated_feed_forward(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, *, activation: str,
                       gate_up_bias: torch.Tensor | None = None, down_bias: torch.Tensor | None = None,
                       residual: torch.Tensor | None = None) -> torch.Tensor:
    """``(act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd (+ residual)`` for ``x`` [T, H],
    ``gate_up`` = [Wg; Wu] [2 I, H] and ``down`` [H, I] in the Hugging Face layout.

    ``activation`` is a name of ``ops.nn.ACT_CODES``. bf16 CUDA rows with H and I
    multiples of 8 run the kernels; every gradient is available (parameters
    with a ``main_grad`` accumulate into it in fp32)."""

    _check(x, gate_up, down, activation, gate_up_bias, down_bias, residual)
    if x.is_cuda and x.dtype == torch.bfloat16 and x.shape[0] > 0 and kernel_widths(x.shape[1], down.shape[1]):
        args = (x, gate_up, down, gate_up_bias, down_bias, residual)
        act = _CODES[activation]
        if torch.is_grad_enabled() and wants_grad(*args):
            if plain(gate_up) and plain(down) and plain(gate_up_bias) and plain(down_bias):
                return ext().gated_ffn_apply(*args, act, status(x.device))
            return GatedFeedForwardFn.apply(*args, act)
        return ext().gated_ffn_forward(x, view(gate_up), view(down), view(gate_up_bias), view(down_bias), residual, act,
                                       False, status(x.device))[0]
    return gated_feed_forward_reference(x, gate_up, down, activation, gate_up_bias, down_bias, residual)


__all__ = ["GatedFeedForwardFn", "gated_feed_forward", "gated_feed_forward_reference", "kernel_widths"]
