"""Log probabilities of given tokens, with entropy and top alternatives, and
their gradient (HIP): an LM's loss, and its scoring.

One pass over the logits where they are, in bfloat16 or float32, with no copy
in float32 and no (tokens, vocabulary) matrix of log probabilities; the
backward reads them once more and writes their gradient.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import ops

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


def cross_entropy(logits: Tensor, targets: Tensor, ignore_index: int = IGNORE) -> Tensor:
    """Mean next-token loss in float32: ``F.cross_entropy`` of the float32 logits
    with class indices (its mean over the targets that are not ignored)."""
    lp = token_logprobs(logits, targets, 0, ignore_index).logprob
    return -lp.sum() / (targets != ignore_index).sum()
