"""A branch's way back into the residual stream, with the norms on both sides of
it (HIP).

With RMS norms, a stream ``x`` and a branch's output ``y``,

    r = x + scale * sigmoid(gate) * post_norm(y),    z = norm(r)

are one pass over the rows: ``r`` is the stream from here on, ``z`` what the next
branch reads.  Each of the post norm, the gate and the scale may be absent.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import ops


class Residual(NamedTuple):
    r: Tensor  # the stream, in x's type
    z: Tensor  # its norm, in y's type


def residual_norm(x: Tensor, y: Tensor, weight: Tensor | None = None, *, post_weight: Tensor | None = None,
                  gate: Tensor | None = None, scale: Tensor | None = None, eps: float = 1e-6) -> Residual:
    """``r = x + scale * sigmoid(gate) * n`` and ``z = r / rms(r) * weight`` over the last
    dimension, with ``n = y / rms(y) * post_weight`` (``y`` itself without a
    ``post_weight``) and ``rms(v) = sqrt(mean(v^2) + eps)``.

    ``x``, ``y``: (..., D) of one shape and type, bfloat16 or float32, or a float32
    stream beside a bfloat16 branch; D up to 8192.  ``gate``: logits, as ``y``.  ``weight``,
    ``post_weight``, ``scale``: (D,), of one type.  Sums are float32; ``z``, and the
    gradients, are computed from ``r`` before it is rounded.  Kept for the backward are ``x``,
    ``y`` and the gate, or for a float32 stream with none of the three parts ``r`` alone.
    """
    ops.ensure()
    r, z, _, _ = torch.ops.gmdn.residual_norm_fwd(x, y, weight, post_weight, gate, scale, eps)
    return Residual(r, z)
