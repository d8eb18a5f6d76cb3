"""Frozen linear weights held in microscaled 4-bit floating point.

``quantize_linears_fp4`` swaps the 2-D linear weights of an encoder for
:class:`FP4Weight` submodules under the same attribute names; the packed-row
linear and feed-forward helpers of ``ops.nn`` dispatch on them, so the encoder
then embeds with 4-bit products (``ops.fp4``). It is a serving transform: the
weights are frozen and no longer export; save or export the model first. Fused
gate / up projections are quantised in their two parts, which the gated
feed-forward kernel needs.

Parity: the weight-swapping entry of src/representax/models/adapters.py:30-267
(``apply_quantized_lora``), for a format that the reference does not have.
"""

from __future__ import annotations

import re

import torch
from torch import nn

from representax_b200.ops.fp4 import BLOCK, FP4Operand, dequantize, quantize

# Attribute names of fused [gate; up] weights.
_GATED = re.compile(r"(^|\.)(gate_up|gate_up_w|Wi)$")
# 2-D parameters that are not linear weights of the towers.
_SKIP = re.compile(r"embed|embeddings\.|\.word$|^word$|position|pos_embed|class_embedding|patch_w$|connector")


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
    """Swap every matching 2-D linear weight of ``model`` for an :class:`FP4Weight` and freeze the rest."""

    pattern = re.compile(target_pattern)
    targets = []
    for mod_name, module in model.named_modules():
        for attr, p in list(module._parameters.items()):
            full = f"{mod_name}.{attr}" if mod_name else attr
            if p is not None and p.ndim == 2 and not _SKIP.search(full) and pattern.search(full):
                targets.append((module, attr, full))
    if not targets:
        raise ValueError(f"no linear weights match target_pattern {target_pattern!r}")
    for p in model.parameters():
        p.requires_grad_(False)
    for module, attr, full in targets:
        weight = module._parameters.pop(attr)
        module.add_module(attr, FP4Weight(weight, fmt=fmt, parts=2 if _GATED.search(full) else 1))
    return model


__all__ = ["FP4Weight", "quantize_linears_fp4"]
