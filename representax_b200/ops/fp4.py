"""Microscaled 4-bit floating point: quantisation, products, and the linear
and gated feed-forward layers over 4-bit operands.

Two formats of E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign):

* ``"mxfp4"``: a power-of-two scale per 32 values of a row,
  ``2^max(-126, ceil(log2(amax / 6)))``, so that no value saturates;
* ``"nvfp4"``: an E4M3 scale per 16 values and a power-of-two factor per row,
  ``f = 2^ceil(log2(rowmax / 2688))``, ``s = E4M3(amax / 6 / f)``.

Roundings are to nearest, ties to even. A block (MXFP4) or row (NVFP4) that
holds an infinity or a NaN is NaN as a whole, and so are products with it.
Scales are kept in the order the tensor core reads (``csrc/fp4.cuh``), so a
product loads them with plain copies. K may be any size: codes are padded with
zeros to whole blocks.

A layer's weight is quantised once (:func:`quantize`, or
``models.fp4.FP4Weight`` inside a model); its activations are quantised inside
every call. bf16 CUDA rows run the kernels, anything else the PyTorch statement.
Weights are frozen: the backward pass gives the gradients of the input
(``dx = dy Q(W)``, the quantiser counted as the identity), bias and residual. A
forward pass gives the same values whether or not a gradient is asked for.

Parity: no counterpart in the reference; the 4-bit sibling of its fp8 linear
(src/representax/precision.py:127-221).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ._ext import ext, status
from .ffn import plain, view, wants_grad
from .functional import _colsum_into, _GradSink

FORMATS = {"mxfp4": 1, "nvfp4": 2}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
_TYPES = frozenset((torch.bfloat16, torch.float16, torch.float32))
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _groups(k: int, fmt: str) -> int:
    return (k + 255) // 256 * (2 if fmt == "mxfp4" else 4)


@dataclass
class FP4Operand:
    """A matrix [rows, k] held in 4 bits.

    ``data`` uint8 [rows, 16 ceil(k / 32)]: two codes a byte, the even column in
    the low nibble. ``scales`` uint8 [parts * ceil(rows / parts / 128), groups, 512].
    ``row_scale`` fp32 [rows] (NVFP4). ``parts`` equal groups of rows (gate and up
    of a fused projection) have scale tiles of their own."""

    data: torch.Tensor
    scales: torch.Tensor
    row_scale: torch.Tensor | None
    fmt: str
    k: int
    parts: int = 1

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def shape(self) -> tuple[int, int]:
        return (self.rows, self.k)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def part(self, index: int) -> "FP4Operand":
        """One of the parts as an operand of its own (views, no copy)."""

        if not 0 <= index < self.parts:
            raise IndexError(f"part {index} of {self.parts}")
        n, t = self.rows // self.parts, self.scales.shape[0] // self.parts
        return FP4Operand(self.data[index * n:(index + 1) * n], self.scales[index * t:(index + 1) * t],
                          None if self.row_scale is None else self.row_scale[index * n:(index + 1) * n], self.fmt, self.k)


def _check_format(fmt: str) -> None:
    if fmt not in FORMATS:
        raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")


def empty_operand(rows: int, k: int, fmt: str, device, parts: int = 1) -> FP4Operand:
    tiles = parts * ((rows // parts + 127) // 128)
    return FP4Operand(torch.empty(rows, (k + 31) // 32 * 16, dtype=torch.uint8, device=device),
                      torch.empty(tiles, _groups(k, fmt), 512, dtype=torch.uint8, device=device),
                      torch.empty(rows, dtype=torch.float32, device=device) if fmt == "nvfp4" else None, fmt, k, parts)


def quantize(x: torch.Tensor, fmt: str = "nvfp4", *, parts: int = 1) -> FP4Operand:
    """``x`` [rows, k] (bf16, fp16 or fp32) in 4 bits, scales along its rows."""

    _check_format(fmt)
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"x must be a matrix with at least one column, got {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if parts < 1 or x.shape[0] % parts:
        raise ValueError(f"{x.shape[0]} rows do not split into {parts} equal parts")
    if not x.is_cuda:
        return _pack_reference(x.detach(), fmt, parts)
    if x.stride(1) != 1:
        x = x.contiguous()
    data, scales, row = ext().fp4_quantize(x, parts, FORMATS[fmt])
    return FP4Operand(data, scales, row, fmt, x.shape[1], parts)


def dequantize(op: FP4Operand, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that ``op`` stands for (exact in bf16 and fp32)."""

    if out is None:
        out = torch.empty(op.rows, op.k, dtype=dtype, device=op.device)
    elif out.shape != op.shape:
        raise ValueError(f"out must be {op.shape}, got {tuple(out.shape)}")
    if not op.data.is_cuda:
        return out.copy_(_unpack_reference(op))
    ext().fp4_dequantize(op.data, op.scales, op.row_scale, op.parts, FORMATS[op.fmt], out)
    return out


def _check_product(a_cols: int, b: FP4Operand, bias, residual, rows: int) -> None:
    if a_cols != b.k:
        raise ValueError(f"the operands contract over {a_cols} and {b.k} values")
    if bias is not None and bias.shape != (b.rows,):
        raise ValueError(f"bias must be [{b.rows}]")
    if residual is not None and residual.shape != (rows, b.rows):
        raise ValueError(f"residual must be [{rows}, {b.rows}]")


def gemm(a: FP4Operand, b: FP4Operand, *, bias: torch.Tensor | None = None,
         residual: torch.Tensor | None = None) -> torch.Tensor:
    """``a b^T (+ bias) (+ residual)`` in bf16 for two operands of one format
    (bf16 ``bias`` [b.rows] and ``residual`` [a.rows, b.rows])."""

    _check_product(a.k, b, bias, residual, a.rows)
    if a.fmt != b.fmt:
        raise ValueError(f"one format a product: got {a.fmt} and {b.fmt}")
    if a.device != b.device:
        raise ValueError(f"operands are on {a.device} and {b.device}")
    if a.parts != 1:
        raise ValueError("the left operand has one part")
    if not a.data.is_cuda:
        y = _unpack_reference(a) @ _unpack_reference(b).T
        y = y if bias is None else y + bias.float()
        return (y if residual is None else y + residual.float()).to(torch.bfloat16)
    return ext().fp4_gemm(a.data, a.scales, a.row_scale, b.data, b.scales, b.row_scale, b.parts, a.k, FORMATS[a.fmt], bias,
                          residual, status(a.device))


def _linear(x, w: FP4Operand, bias, residual):
    return ext().fp4_linear(x if x.stride(1) == 1 else x.contiguous(), w.data, w.scales, w.row_scale, w.parts,
                            FORMATS[w.fmt], None if bias is None else view(bias).contiguous(), residual,
                            status(x.device))


def _dgrad(dy, w: FP4Operand):
    return ext().fp4_linear_dgrad(dy, w.data, w.scales, w.row_scale, w.parts, w.k, FORMATS[w.fmt], status(dy.device))


def _bias_gradient(dy, bias):
    sink = _GradSink(bias)
    if dy.shape[0] and dy.shape[1] % 8 == 0 and dy.is_contiguous() and dy.data_ptr() % 16 == 0:
        _colsum_into(dy, sink)
    else:
        sink.buffer().add_(dy.float().sum(0))
    return sink.result()


class LinearFP4Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual):
        ctx.weight = weight
        ctx.save_for_backward(bias)
        return _linear(x, weight, bias, residual)

    @staticmethod
    def backward(ctx, dy):
        (bias,) = ctx.saved_tensors
        w = ctx.weight
        dx = db = None
        if ctx.needs_input_grad[0]:
            dx = _dgrad(dy, w)
        if ctx.needs_input_grad[2]:
            db = _bias_gradient(dy, bias)
        return dx, None, db, dy if ctx.needs_input_grad[3] else None


def linear_fp4(x: torch.Tensor, weight: FP4Operand, bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``Q(x) Q(W)^T (+ bias) (+ residual)`` for ``x`` [T, K] and a weight from :func:`quantize`."""

    if x.dim() != 2:
        raise ValueError(f"x must be a matrix, got {tuple(x.shape)}")
    _check_product(x.shape[1], weight, bias, residual, x.shape[0])
    if x.device != weight.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    if x.is_cuda and x.dtype == torch.bfloat16:
        if residual is not None and residual.dtype != torch.bfloat16:
            raise TypeError("residual must be bfloat16 like x")
        if torch.is_grad_enabled() and wants_grad(x, bias, residual):
            if plain(bias) and x.stride(1) == 1 and (bias is None or bias.is_contiguous()):
                return ext().fp4_linear_apply(x, weight.data, weight.scales, weight.row_scale, weight.parts,
                                              FORMATS[weight.fmt], bias, residual, status(x.device))
            return LinearFP4Fn.apply(x, weight, bias, residual)
        return _linear(x, weight, bias, residual)
    return linear_fp4_reference(x, weight, bias, residual)


def _feed_forward(x, gate_up: FP4Operand, down: FP4Operand, activation, gate_up_bias, down_bias, residual):
    from .nn import ACT_CODES

    bias = lambda t: None if t is None else view(t).contiguous()  # noqa: E731
    return ext().fp4_ffn(x if x.stride(1) == 1 else x.contiguous(), gate_up.data, gate_up.scales, gate_up.row_scale,
                         FORMATS[gate_up.fmt], down.data, down.scales, down.row_scale, FORMATS[down.fmt],
                         ACT_CODES[activation], bias(gate_up_bias), bias(down_bias), residual, status(x.device))


class GatedFeedForwardFP4Fn(torch.autograd.Function):
    """The block's own forward, so that a value does not depend on whether its gradient is asked for. The backward
    runs the first product once more (z in bf16) instead of keeping [T, 2 I] values of it."""

    @staticmethod
    def forward(ctx, x, gate_up, down, activation, gate_up_bias, down_bias, residual):
        ctx.weights, ctx.activation = (gate_up, down), activation
        ctx.save_for_backward(x, gate_up_bias, down_bias)
        return _feed_forward(x, gate_up, down, activation, gate_up_bias, down_bias, residual)

    @staticmethod
    def backward(ctx, dy):
        from .nn import gated_activation

        x, gate_up_bias, down_bias = ctx.saved_tensors
        gate_up, down = ctx.weights
        need = ctx.needs_input_grad
        dx = db1 = db2 = None
        if need[0] or need[4]:
            if dy.shape[0]:
                z = _linear(x, gate_up, gate_up_bias, None).requires_grad_()
                with torch.enable_grad():
                    h = gated_activation(z, ctx.activation)
                (dz,) = torch.autograd.grad(h, z, _dgrad(dy, down))
            else:
                dz = dy.new_zeros(0, gate_up.rows)
            dx = _dgrad(dz, gate_up) if need[0] else None
            db1 = _bias_gradient(dz, gate_up_bias) if need[4] else None
        if need[5]:
            db2 = _bias_gradient(dy, down_bias)
        return dx, None, None, None, db1, db2, dy if need[6] else None


def gated_feed_forward_fp4(x: torch.Tensor, gate_up: FP4Operand, down: FP4Operand, *, activation: str,
                           gate_up_bias: torch.Tensor | None = None, down_bias: torch.Tensor | None = None,
                           residual: torch.Tensor | None = None) -> torch.Tensor:
    """The gated feed-forward block over 4-bit operands.

    ``h = act(Q(x) Q(Wg)^T + bg) * (Q(x) Q(Wu)^T + bu)``, ``y = Q(h) Q(Wd)^T + bd
    (+ residual)``; ``gate_up`` is quantised with ``parts=2``. In MXFP4 the first
    product's kernel quantises its fp32 results itself (h is never written in 16
    bits); in NVFP4, whose row factor needs the whole row, h passes through the type of x.
    Gradients of x, the biases and the residual (both quantisers counted as the identity)."""

    from .nn import ACT_CODES

    if activation not in ACT_CODES:
        raise ValueError(f"unsupported activation {activation!r}")
    if gate_up.parts != 2:
        raise ValueError("gate_up must be quantised with parts=2")
    if x.dim() != 2 or gate_up.rows != 2 * down.k:
        raise ValueError(f"gate_up must be [2 I, H] and down [H', I]: got {gate_up.shape} and {down.shape}")
    _check_product(x.shape[1], gate_up, gate_up_bias, None, x.shape[0])
    _check_product(down.k, down, down_bias, residual, x.shape[0])
    if not x.device == gate_up.device == down.device:
        raise ValueError(f"x is on {x.device}, the weights on {gate_up.device} and {down.device}")
    if not (x.is_cuda and x.dtype == torch.bfloat16):
        return gated_feed_forward_fp4_reference(x, gate_up, down, activation, gate_up_bias, down_bias, residual)
    if residual is not None and residual.dtype != torch.bfloat16:
        raise TypeError("residual must be bfloat16 like x")
    if torch.is_grad_enabled() and wants_grad(x, gate_up_bias, down_bias, residual):
        return GatedFeedForwardFP4Fn.apply(x, gate_up, down, activation, gate_up_bias, down_bias, residual)
    return _feed_forward(x, gate_up, down, activation, gate_up_bias, down_bias, residual)


# ------------------------------------------------------------ PyTorch statement
def _pow2_ceil(v: torch.Tensor) -> torch.Tensor:
    mantissa, exponent = torch.frexp(v)
    e = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(min=-126)
    return torch.where(v > 0, torch.ldexp(torch.ones_like(v), e), torch.ones_like(v))


def quantize_reference(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """(codes as signed E2M1 values [R, blocks, B], block scales [R, blocks], row factors [R] or None) in fp32."""

    _check_format(fmt)
    size = BLOCK[fmt]
    xf = x.float()
    r, c = xf.shape
    b = torch.nn.functional.pad(xf, (0, -c % size)).reshape(r, -1, size)
    amax = b.abs().amax(-1)
    six = torch.full_like(amax, 6.0)
    row = None
    nan = torch.full((), float("nan"), device=x.device)
    if fmt == "mxfp4":
        # ceil(log2(amax / 6)) from amax = m 2^e, 0.5 <= m < 1: e - 3 for m <= 0.75, e - 2 above
        mantissa, exponent = torch.frexp(amax)
        e = torch.where(mantissa <= 0.75, exponent - 3, exponent - 2).clamp(min=-126)
        scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.ones_like(amax))
        scale = torch.where(amax.isfinite(), scale, nan)
        full = scale
    else:
        top = amax.amax(1) if amax.shape[1] else amax.sum(1)
        row = torch.where(top.isfinite(), _pow2_ceil(top / torch.full_like(top, 2688.0)), nan)
        scale = (amax / six / row[:, None]).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        full = scale * row[:, None]
    ok = full > 0
    q = torch.where(ok[..., None], b / torch.where(ok, full, torch.ones_like(full))[..., None], torch.zeros_like(b))
    mag = q.abs().clamp(max=6.0)
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    return torch.copysign(torch.round(mag / step) * step, q), scale, row


def fake_quantize_reference(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """The fp32 values of ``x`` after a round trip through 4 bits."""

    q, scale, row = quantize_reference(x, fmt)
    v = q * scale[..., None]
    if row is not None:
        v = v * row[:, None, None]
    return v.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _product_reference(x, weight: FP4Operand, bias, residual):
    """Q(x) Q(W)^T (+ bias) (+ residual) in fp32 for fp32 ``x``."""

    y = fake_quantize_reference(x, weight.fmt)
    y = x + (y - x).detach()  # the quantiser counts as the identity in the backward pass (the sum is exact)
    y = y @ _unpack_reference(weight).to(y.device).T
    y = y if bias is None else y + bias.float()
    return y if residual is None else y + residual.float()


def linear_fp4_reference(x, weight: FP4Operand, bias=None, residual=None):
    return _product_reference(x.float(), weight, bias, residual).to(x.dtype)


def gated_feed_forward_fp4_reference(x, gate_up: FP4Operand, down: FP4Operand, activation, gate_up_bias=None, down_bias=None,
                                     residual=None):
    """The block in fp32, rounded where the kernels round: h to the type of ``x`` unless both formats are MXFP4, y once."""

    from .nn import _act_reference

    z = _product_reference(x.float(), gate_up, gate_up_bias, None)
    h = _act_reference(z[:, :down.k], activation) * z[:, down.k:]
    if gate_up.fmt != "mxfp4" or down.fmt != "mxfp4":
        h = h.to(x.dtype).float()
    return _product_reference(h, down, down_bias, residual).to(x.dtype)


def _pack_reference(x: torch.Tensor, fmt: str, parts: int) -> FP4Operand:
    q, scale, row = quantize_reference(x, fmt)
    op = empty_operand(x.shape[0], x.shape[1], fmt, x.device, parts)
    values = torch.tensor(E2M1, device=x.device)
    codes = torch.searchsorted(values, q.abs()).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    codes = codes.reshape(x.shape[0], -1)
    codes = torch.nn.functional.pad(codes, (0, 2 * op.data.shape[1] - codes.shape[1])).reshape(x.shape[0], -1, 2)
    op.data.copy_(codes[..., 0] | (codes[..., 1] << 4))
    if fmt == "mxfp4":
        mantissa, exponent = torch.frexp(scale)
        bytes_ = torch.where(scale.isfinite(), exponent - 1 + 127, 255).to(torch.uint8)
        filler = 127
    else:
        bytes_ = scale.to(torch.float8_e4m3fn).view(torch.uint8)
        filler = 0
        op.row_scale.copy_(row)
    # [parts, tiles, q = 4, l = 32, groups, 4] -> [parts * tiles, groups, l, q, 4]
    n = x.shape[0] // parts
    tiles, groups = (n + 127) // 128, op.scales.shape[1]
    grid = torch.zeros(parts, tiles * 128, groups * 4, dtype=torch.uint8, device=x.device)
    grid[:, :n] = filler
    grid[:, :n, :bytes_.shape[1]] = bytes_.reshape(parts, n, -1)
    grid = grid.reshape(parts * tiles, 4, 32, groups, 4).permute(0, 3, 2, 1, 4)
    op.scales.copy_(grid.reshape(parts * tiles, groups, 512))
    return op


def scale_values(op: FP4Operand) -> torch.Tensor:
    """Block scales [rows, blocks] (fp32) of an operand, in row order."""

    tiles, groups, _ = op.scales.shape
    grid = op.scales.reshape(tiles, groups, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(op.parts, -1, groups * 4)
    n, blocks = op.rows // op.parts, -(-op.k // BLOCK[op.fmt])
    grid = grid[:, :n, :blocks].reshape(op.rows, blocks)
    if op.fmt == "nvfp4":
        return grid.contiguous().view(torch.float8_e4m3fn).float()
    scale = torch.ldexp(torch.ones(grid.shape, device=grid.device), grid.int() - 127)
    return torch.where(grid == 255, torch.full_like(scale, float("nan")), scale)


def _unpack_reference(op: FP4Operand) -> torch.Tensor:
    codes = torch.stack((op.data & 0x0F, op.data >> 4), dim=-1).reshape(op.rows, -1)[:, :op.k]
    values = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=op.device)[codes.long()]
    scale = scale_values(op).repeat_interleave(BLOCK[op.fmt], dim=1)[:, :op.k]
    v = values * scale
    return v if op.row_scale is None else v * op.row_scale[:, None]


__all__ = ["BLOCK", "FORMATS", "FP4Operand", "GatedFeedForwardFP4Fn", "LinearFP4Fn", "dequantize",
           "fake_quantize_reference", "gated_feed_forward_fp4", "gated_feed_forward_fp4_reference", "gemm", "linear_fp4",
           "linear_fp4_reference", "quantize", "quantize_reference", "scale_values"]
