"""Gated feed-forward block of the decoder and encoder layers.

``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual`` on packed
token rows, with the gate and up projections in one weight ``[Wg; Wu]``.

bf16 CUDA rows run hand-written kernels: one launch computes both
projections, the activation and the product (``csrc/gated.cu``; up to
``FEW_ROWS`` rows the weight-streaming kernel of ``csrc/few_rows.cu``), a second
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

from . import gemm as G
from ._ext import ext, status
from .functional import _colsum_into, _GradSink, compute_view

# Most rows that the weight-streaming kernel takes.
FEW_ROWS = 64


def _codes() -> dict[str, int]:
    from .nn import ACT_CODES

    return ACT_CODES


def rows16(t: torch.Tensor) -> torch.Tensor:
    """``t`` with 16-byte aligned rows of unit inner stride, as the tensor maps
    need them (a copy only where it is not)."""

    if (t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _vector16(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check(x, gate_up, down, activation, gate_up_bias, down_bias, residual) -> None:
    if activation not in _codes():
        raise ValueError(f"unsupported activation {activation!r}")
    if x.dim() != 2 or gate_up.dim() != 2 or down.dim() != 2:
        raise ValueError("x, gate_up and down must be matrices")
    width = down.shape[1]
    if tuple(gate_up.shape) != (2 * width, x.shape[1]) or down.shape[0] != x.shape[1]:
        raise ValueError(f"gate_up must be [2 I, H] and down [H, I] for x [T, H]: got {tuple(gate_up.shape)}, "
                         f"{tuple(down.shape)} and {tuple(x.shape)}")
    if gate_up_bias is not None and tuple(gate_up_bias.shape) != (2 * width,):
        raise ValueError(f"gate_up_bias must be [{2 * width}]")
    if down_bias is not None and tuple(down_bias.shape) != (down.shape[0],):
        raise ValueError(f"down_bias must be [{down.shape[0]}]")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have the shape and type of x")
    for name, t in (("gate_up", gate_up), ("down", down), ("gate_up_bias", gate_up_bias), ("down_bias", down_bias),
                    ("residual", residual)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")


def _project_down(h, w, bias, residual):
    if h.shape[0] <= FEW_ROWS:
        y = torch.empty(h.shape[0], w.shape[0], dtype=torch.bfloat16, device=h.device)
        ext().few_rows_linear(h, w, 1, 0, bias, residual, y, status(h.device))
        return y
    return G.linear_forward(h, w, bias, residual=residual)


class GatedFeedForwardFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_up, down, gate_up_bias, down_bias, residual, act):
        C, dev = ext(), x.device
        x = rows16(x)
        w1, w2 = rows16(compute_view(gate_up)), rows16(compute_view(down))
        b1 = None if gate_up_bias is None else _vector16(compute_view(gate_up_bias))
        b2 = None if down_bias is None else _vector16(compute_view(down_bias))
        rows, width = x.shape[0], w2.shape[1]
        h = torch.empty(rows, width, dtype=torch.bfloat16, device=dev)
        need_z = any(ctx.needs_input_grad[i] for i in (0, 1, 3))  # a gradient that goes through dz
        saved = exps = None
        if need_z:
            saved = torch.empty(rows, 2 * width, dtype=torch.float16, device=dev)
            exps = torch.empty(rows, (width + 31) // 32, dtype=torch.int16, device=dev)
        if rows <= FEW_ROWS and not need_z:
            C.few_rows_linear(x, w1, 2, act, b1, None, h, status(dev))
        else:
            C.gated_forward(x, w1, b1, h, saved, exps, act, status(dev))
        y = _project_down(h, w2, b2, None if residual is None else rows16(residual))
        empty = torch.empty(0, device=dev)
        opt = lambda t: empty if t is None else t  # noqa: E731
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else empty, gate_up, down,
                              h if ctx.needs_input_grad[2] else empty, opt(saved), opt(exps), opt(gate_up_bias),
                              opt(down_bias))
        ctx.biases = (gate_up_bias is not None, down_bias is not None)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gate_up, down, h, saved, exps, b1, b2 = ctx.saved_tensors
        need = ctx.needs_input_grad
        dres = dy if need[5] else None
        dy = rows16(dy)
        dx = None
        s1, s2 = _GradSink(gate_up), _GradSink(down)
        sb1 = _GradSink(b1) if ctx.biases[0] else None
        sb2 = _GradSink(b2) if ctx.biases[1] else None
        if need[2]:
            G.linear_wgrad(dy, h, s2.buffer())
        if sb2 is not None:
            _colsum_into(dy, sb2)
        if need[0] or need[1] or need[3]:
            dz = torch.empty(dy.shape[0], gate_up.shape[0], dtype=torch.bfloat16, device=dy.device)
            ext().gated_backward(dy, rows16(compute_view(down)), saved, exps, dz, status(dy.device))
            if need[1]:
                G.linear_wgrad(dz, x, s1.buffer())
            if sb1 is not None:
                _colsum_into(dz, sb1)
            if need[0]:
                dx = G.linear_dgrad(dz, rows16(compute_view(gate_up)))
        return (dx, s1.result(), s2.result(), sb1.result() if sb1 is not None else None,
                sb2.result() if sb2 is not None else None, dres, None)


def gated_feed_forward_reference(x, gate_up, down, activation, gate_up_bias=None, down_bias=None, residual=None):
    """The block in fp32, rounded once to the type of ``x``."""

    from .nn import _act_reference

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
    if x.is_cuda and x.dtype == torch.bfloat16 and x.shape[0] > 0 and x.shape[1] % 8 == 0 and down.shape[1] % 8 == 0:
        return GatedFeedForwardFn.apply(x, gate_up, down, gate_up_bias, down_bias, residual, _codes()[activation])
    return gated_feed_forward_reference(x, gate_up, down, activation, gate_up_bias, down_bias, residual)


__all__ = ["FEW_ROWS", "GatedFeedForwardFn", "gated_feed_forward", "gated_feed_forward_reference"]
