"""Layer norm over the last dimension, with its backward pass (HIP).

``layer_norm`` is ``torch.nn.functional.layer_norm`` over one dimension of up
to 16384 values, on bfloat16 or float32 GPU tensors, with two things beside:
the output may be bfloat16 where the input is float32 (a float32 residual
stream into a bfloat16 projection, without a copy between), and the input may
be kept for the backward in 8 bits (``checkpoint="int8"``; gmdn_amd.act8 has
the format).  Statistics and sums are float32; the gradients of weight and
bias are summed in a fixed order.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from . import ops


def checked_checkpoint(checkpoint: str | None) -> bool:
    """Whether activations are kept in 8 bits; refuses any other name."""
    if checkpoint not in (None, "int8"):
        raise ValueError(f"checkpoint is None or 'int8', got {checkpoint!r}")
    return checkpoint == "int8"


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5, *,
               dtype: torch.dtype | None = None, checkpoint: str | None = None) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    ``x``: (..., D) bfloat16 or float32.  ``weight``, ``bias``: (D,), both
    bfloat16 or both float32; a bias needs a weight.  ``dtype``: the output's,
    by default ``x``'s; bfloat16 beside a float32 ``x`` is the one other pair.
    ``checkpoint="int8"`` keeps ``x`` for the backward in 8 bits: a quarter of
    float32's memory, and gradients that see each value of ``x`` within 1 / 254
    of its group's largest magnitude.
    """
    ops.ensure()
    pack = checked_checkpoint(checkpoint) and ops.wants_grad(x, weight, bias)
    return torch.ops.gmdn.layer_norm_fwd(x, weight, bias, eps, dtype or x.dtype, pack)[0]


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension through ``layer_norm``.  Under
    bfloat16 autocast the output is bfloat16, as the products that follow it
    take it."""

    def __init__(self, dim: int, eps: float = 1e-5, checkpoint: str | None = None, bias: bool = True):
        super().__init__(dim, eps=eps, bias=bias)
        checked_checkpoint(checkpoint)
        self.checkpoint = checkpoint

    def output_dtype(self, x: Tensor) -> torch.dtype:
        auto = torch.is_autocast_enabled(x.device.type) and \
            torch.get_autocast_dtype(x.device.type) == torch.bfloat16
        return torch.bfloat16 if auto else x.dtype

    def forward(self, x: Tensor) -> Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps, dtype=self.output_dtype(x), checkpoint=self.checkpoint)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, checkpoint={self.checkpoint}"
