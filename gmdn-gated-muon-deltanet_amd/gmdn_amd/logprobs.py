"""Log probabilities of given tokens, with entropy and top alternatives, and
their gradient (HIP): an LM's loss, and its scoring.

One pass over the logits where they are, in bfloat16 or float32, with no copy
in float32 and no (tokens, vocabulary) matrix of log probabilities; the
backward reads them once more and writes their gradient.  ``linear_logprobs``
takes the hidden states and the head's weight instead, and never has the logits
in memory.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import ops, scan

IGNORE = -100
MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """Per position (the logits' leading dimensions), float32:"""

    logprob: Tensor        # of the given token
    entropy: Tensor        # of the distribution, in nats
    top_logprobs: Tensor   # (..., top), largest first
    top_tokens: Tensor     # (..., top), int64


def token_logprobs(logits: Tensor, tokens: Tensor, top: int = 0, ignore_index: int = IGNORE) -> TokenLogprobs:
    """``log_softmax(logits)`` at ``tokens``, the distribution's entropy, and its
    ``top`` (at most 32) likeliest tokens, equal ones in the order of their index.

    ``logits``: (..., V) bfloat16 or float32, read in place also as a slice of
    a padded vocabulary.  ``tokens``: (...) integers; ``ignore_index`` gives log
    probability 0 without a gradient, any other token outside [0, V) NaN.
    Masked logits are ``-inf``; a row of nothing else has log probabilities
    ``-inf``, entropy 0 and no gradient.  Differentiable through ``logprob``,
    ``entropy`` and ``top_logprobs``.
    """
    ops.ensure()
    lp, entropy, top_lp, top_tokens, _ = torch.ops.gmdn.logprobs_fwd(logits, tokens, top, ignore_index)
    return TokenLogprobs(lp, entropy, top_lp, top_tokens)


class LinearLogprobs(NamedTuple):
    """Per position (the hidden states' leading dimensions), float32:"""

    logprob: Tensor  # of the given token
    entropy: Tensor  # of the distribution, in nats


def linear_logprobs(x: Tensor, weight: Tensor, tokens: Tensor, ignore_index: int = IGNORE,
                    precision: str | None = None) -> LinearLogprobs:
    """``token_logprobs(x @ weight.t(), tokens)`` without the logits: they are
    formed tile by tile, and again a piece of the vocabulary at a time in the backward.

    ``x``: (..., D) hidden states, ``weight``: (V, D), both bfloat16 or both float32
    (under autocast they are taken in its type, as by a linear layer).  The logits are
    float32 sums that are not rounded; their gradient is rounded to bfloat16 beside
    bfloat16 operands.  float32 products are taken as three products of bfloat16
    pieces, about 2^-16 relative error each, or in 'ieee' as six, which leave float32's
    rounding; ``precision`` ('tf32' or 'ieee') overrides the process-wide setting
    (``set_precision``).  Tokens are treated as in
    ``token_logprobs``: one outside the vocabulary is NaN, and through its log probability
    ``weight``'s gradient, which sums over all rows.  Differentiable through both outputs, in ``x``
    and ``weight``.
    """
    ops.ensure()
    dt = ops.autocast_dtype(x)
    if dt is not None:
        x, weight = x.to(dt), weight.to(dt)
    lp, entropy, _ = torch.ops.gmdn.linear_logprobs_fwd(x, weight, tokens, ignore_index,
                                                        scan.precision_code(precision))
    return LinearLogprobs(lp, entropy)


def _mean_loss(logprob: Tensor, targets: Tensor, ignore_index: int) -> Tensor:
    return -logprob.sum() / (targets != ignore_index).sum()


def linear_cross_entropy(x: Tensor, weight: Tensor, targets: Tensor, ignore_index: int = IGNORE,
                         precision: str | None = None) -> Tensor:
    """``cross_entropy(x @ weight.t(), targets)`` without the logits."""
    return _mean_loss(linear_logprobs(x, weight, targets, ignore_index, precision).logprob, targets, ignore_index)


def cross_entropy(logits: Tensor, targets: Tensor, ignore_index: int = IGNORE) -> Tensor:
    """Mean next-token loss in float32: ``F.cross_entropy`` of the float32 logits
    with class indices (its mean over the targets that are not ignored)."""
    return _mean_loss(token_logprobs(logits, targets, 0, ignore_index).logprob, targets, ignore_index)
