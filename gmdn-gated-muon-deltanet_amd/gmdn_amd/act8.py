"""Activation checkpoints in 8 bits, and the passes that use them (HIP).

What a training step keeps between its passes is mostly activations.  Here
they are kept as int8 values with one float32 scale for each 128 consecutive
values of a row, 1.03 bytes a value:

    scale = amax / 127,  q = rint(x / scale),  x' = q scale

(``amax`` the group's largest magnitude), so ``|x' - x| <= amax / 254``.  A
group below 2^-100 reads back as zeros; one that holds an infinity or a NaN
reads back as NaN.

The forward's outputs are computed from the activations themselves; only the
backward sees the checkpoints.  A call without gradients makes none, and one
with frozen weights none that only they would want.

* ``pack`` / ``unpack`` -- a checkpoint of any tensor.
* ``gelu``     -- GELU that keeps its input in 8 bits.
* ``linear``   -- a linear layer that keeps its input in 8 bits.
* ``mlp``      -- linear, GELU, linear: keeps its input and the hidden layer
  before GELU, 5 bytes a channel of the input where torch's modules under
  bfloat16 keep 18.
* ``norm_mlp`` -- layer norm and the same: the norm's input serves both the
  norm's gradient and, normed again, the first weight's.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch import Tensor

from . import ops


class Packed(NamedTuple):
    """A checkpoint: int8 values in the tensor's shape, and the scale of each
    128 of a row."""

    q: Tensor
    scale: Tensor


def pack(x: Tensor) -> Packed:
    """The 8-bit checkpoint of ``x`` (..., D), bfloat16 or float32."""
    ops.ensure()
    return Packed(*torch.ops.gmdn.act8_pack(x))


def unpack(packed: Packed, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """What the checkpoint reads back as, in ``dtype``."""
    ops.ensure()
    return torch.ops.gmdn.act8_unpack(packed[0], packed[1], dtype)


def gelu(h: Tensor) -> Tensor:
    """GELU (``h`` times the normal distribution function of ``h``), keeping
    ``h`` in 8 bits for the backward."""
    ops.ensure()
    return torch.ops.gmdn.gelu8_fwd(h, ops.wants_grad(h))[0]


def _cast(*tensors: Tensor | None):
    """Under autocast, the tensors in its type (as torch's own products take
    them); differentiable."""
    dev = tensors[0].device.type
    if not torch.is_autocast_enabled(dev):
        return tensors
    dt = torch.get_autocast_dtype(dev)
    return tuple(t if t is None else t.to(dt) for t in tensors)


def _flat(t: Tensor) -> Tensor:
    return t.reshape(-1, t.shape[-1])


def _kept(x: Tensor, wanted: bool):
    """The checkpoint of a product's input, where the weight wants its gradient."""
    return torch.ops.gmdn.act8_pack(x) if wanted else (None, None)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(*_kept(x, ctx.needs_input_grad[1]), weight)
        ctx.has_bias = bias is not None
        return F.linear(x, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        q, scale, weight = ctx.saved_tensors
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = dy @ weight
        if ctx.needs_input_grad[1]:
            x = torch.ops.gmdn.act8_unpack(q, scale, dy.dtype)
            dw = _flat(dy).t() @ _flat(x)
        if ctx.has_bias and ctx.needs_input_grad[2]:
            db = _flat(dy).sum(0)
        return dx, dw, db


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None) -> Tensor:
    """``F.linear`` that keeps ``x`` in 8 bits for the weight's gradient."""
    ops.ensure()
    x, weight, bias = _cast(x, weight, bias)
    if not ops.wants_grad(x, weight, bias):
        return F.linear(x, weight, bias)
    return _Linear.apply(x, weight, bias)


def _mlp_forward(y, w1, w2, pack=True):
    """linear, GELU, linear; returns the output and the hidden checkpoint."""
    h = F.linear(y, w1)
    a, qh, sh = torch.ops.gmdn.gelu8_fwd(h, pack)
    return F.linear(a, w2), qh, sh


def _mlp_backward(dout, qh, sh, w1, w2, need_y, need1, need2, input_again):
    """(dy, dw1, dw2) of linear, GELU, linear, None where not needed;
    ``input_again`` gives the input from its checkpoint, where the first weight
    wants its gradient."""
    da = dout @ w2
    dh, a = torch.ops.gmdn.gelu8_bwd(da, qh, sh, need2)
    del da
    dw2 = _flat(dout).t() @ _flat(a) if need2 else None
    del a
    dw1 = _flat(dh).t() @ _flat(input_again()) if need1 else None
    return dh @ w1 if need_y else None, dw1, dw2


class _Mlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2):
        out, qh, sh = _mlp_forward(x, w1, w2)
        ctx.save_for_backward(*_kept(x, ctx.needs_input_grad[1]), qh, sh, w1, w2)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, scale, qh, sh, w1, w2 = ctx.saved_tensors
        return _mlp_backward(dout, qh, sh, w1, w2, *ctx.needs_input_grad,
                             lambda: torch.ops.gmdn.act8_unpack(q, scale, dout.dtype))


def mlp(x: Tensor, w1: Tensor, w2: Tensor) -> Tensor:
    """``F.linear(F.gelu(F.linear(x, w1)), w2)``, keeping ``x`` and the hidden
    layer in 8 bits."""
    ops.ensure()
    x, w1, w2 = _cast(x, w1, w2)
    if not ops.wants_grad(x, w1, w2):
        return _mlp_forward(x, w1, w2, False)[0]
    return _Mlp.apply(x, w1, w2)


class _NormMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, w1, w2, eps):
        # all but the second weight's gradient want the norm's input again
        pack = any(ctx.needs_input_grad[:4])
        y, mean, rstd, q, scale = torch.ops.gmdn.layer_norm_fwd(x, weight, bias, eps, w1.dtype, pack)
        out, qh, sh = _mlp_forward(y, w1, w2)
        ctx.save_for_backward(*((q, scale, mean, rstd) if pack else (None,) * 4), qh, sh, weight, bias, w1, w2)
        ctx.x_dtype = x.dtype
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, scale, mean, rstd, qh, sh, weight, bias, w1, w2 = ctx.saved_tensors
        need_norm = any(ctx.needs_input_grad[:3])
        dy, dw1, dw2 = _mlp_backward(
            dout, qh, sh, w1, w2, need_norm, *ctx.needs_input_grad[3:5],
            lambda: torch.ops.gmdn.layer_norm8_rebuild(q, scale, weight, bias, mean, rstd, dout.dtype))
        if not need_norm:
            return None, None, None, dw1, dw2, None
        dx, dweight, dbias = torch.ops.gmdn.layer_norm8_bwd(dy, q, scale, weight, mean, rstd, ctx.x_dtype)
        return (dx, dweight if weight is not None else None, dbias if bias is not None else None, dw1, dw2, None)


def norm_mlp(x: Tensor, weight: Tensor | None, bias: Tensor | None, w1: Tensor, w2: Tensor, eps: float = 1e-5) -> Tensor:
    """``mlp(layer_norm(x, weight, bias), w1, w2)``, keeping ``x`` and the
    hidden layer in 8 bits."""
    ops.ensure()
    w1, w2 = _cast(w1, w2)
    if not ops.wants_grad(x, weight, bias, w1, w2):
        return _mlp_forward(torch.ops.gmdn.layer_norm_fwd(x, weight, bias, eps, w1.dtype, False)[0], w1, w2, False)[0]
    return _NormMlp.apply(x, weight, bias, w1, w2, eps)
