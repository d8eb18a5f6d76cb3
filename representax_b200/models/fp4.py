"""Frozen linear weights held in microscaled 4-bit floating point.

``quantize_linears_fp4`` swaps linear weights of an encoder for
:class:`FP4Weight` submodules under the same attribute names; the packed-row
linear and feed-forward helpers of ``ops.nn`` dispatch on them, so the encoder
then embeds with 4-bit products (``ops.fp4``). It is a serving transform: the
weights are frozen and no longer export; save or export the model first.

Only weights that reach nothing but those helpers can be swapped. A module says
which by a class attribute ``packed_linears``: attribute name -> parts of its
rows (2 for a fused gate / up projection, whose halves the gated feed-forward
kernel needs apart). The Qwen3, Qwen3-VL, Qwen2.5-Omni, ModernVBERT and CLIP layers have one.
Everything else (embeddings, lookup tables, patch projections, heads, LoRA
factors, the BERT and MPNet blocks) keeps its weights; a model without such layers is refused.

Parity: the weight-swapping entry of src/representax/models/adapters.py:30-267
(``apply_quantized_lora``), for a format that the reference does not have.
"""

from __future__ import annotations

import re

import torch
from torch import nn

from representax_b200.ops.fp4 import BLOCK, FP4Operand, dequantize, quantize


class FP4Weight(nn.Module):
    """A frozen [out, in] weight in ``"mxfp4"`` or ``"nvfp4"``."""

    def __init__(self, weight: torch.Tensor, *, fmt: str = "nvfp4", parts: int = 1) -> None:
        super().__init__()
        if fmt not in BLOCK:
            raise ValueError(f"fmt must be one of {sorted(BLOCK)}, got {fmt!r}")
        op = quantize(weight.detach(), fmt, parts=parts)
        self.register_buffer("data", op.data)
        self.register_buffer("scales", op.scales)
        self.register_buffer("row_scale", op.row_scale)
        self.fmt, self.parts, self.input_size = fmt, parts, op.k
        self.shape = (op.rows, op.k)

    @property
    def operand(self) -> FP4Operand:
        return FP4Operand(self.data, self.scales, self.row_scale, self.fmt, self.input_size, self.parts)

    def dequantized(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return dequantize(self.operand, dtype)

    def _apply(self, fn, recurse=True):
        """Moves between devices; the row factors stay fp32 under dtype casts."""

        row = self.row_scale
        super()._apply(fn, recurse)
        if row is not None and self.row_scale.dtype != torch.float32:
            self.row_scale = row.to(self.row_scale.device)
        return self


def quantize_linears_fp4(model: nn.Module, *, fmt: str = "nvfp4", target_pattern: str = ".*") -> nn.Module:
    """Swap every matching linear weight of ``model``'s packed-row layers for an :class:`FP4Weight` and freeze the rest.

    The model is changed only after every weight has been quantised, so a
    refusal leaves it as it was."""

    if fmt not in BLOCK:
        raise ValueError(f"fmt must be one of {sorted(BLOCK)}, got {fmt!r}")
    pattern = re.compile(target_pattern)
    able = []
    for mod_name, module in model.named_modules():
        for attr, parts in getattr(type(module), "packed_linears", {}).items():
            if module._parameters.get(attr) is not None:
                able.append((module, attr, f"{mod_name}.{attr}" if mod_name else attr, parts))
    if not able:
        raise ValueError(f"{type(model).__name__} has no linear weights that run on packed rows in 4 bits")
    targets = [t for t in able if pattern.search(t[2])]
    if not targets:
        raise ValueError(f"no linear weights match target_pattern {target_pattern!r}")
    swapped = [FP4Weight(module._parameters[attr], fmt=fmt, parts=parts) for module, attr, _, parts in targets]
    for p in model.parameters():
        p.requires_grad_(False)
    for (module, attr, _, _), weight in zip(targets, swapped):
        del module._parameters[attr]
        module.add_module(attr, weight)
    return model


__all__ = ["FP4Weight", "quantize_linears_fp4"]
