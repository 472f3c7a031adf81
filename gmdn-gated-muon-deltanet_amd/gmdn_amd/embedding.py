"""Token embedding with a scale, and its gradient by sorted tokens (HIP).

``embedding`` is ``scale * weight[tokens]``.  Its gradient is the whole table's,
in one pass over the rows of the cotangent: positions are sorted by token and
each token's rows are summed in float32 in the order of their positions, rounded
once, so that every run gives the same bits; rows that no token names are zeros.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from . import ops


def embedding(tokens: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: int | None = None) -> Tensor:
    """``scale * weight[tokens]``: (..., D) from tokens (...), int64 or int32.

    ``weight``: (V, D) bfloat16 or float32.  A token outside [0, V) gives a row of
    NaN and no gradient.  ``padding_idx`` (negative: from the end): a row that
    is looked up like the others and gets no gradient.
    """
    ops.ensure()
    pad = -1
    if padding_idx is not None:
        vocab = weight.shape[0]
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"padding_idx {padding_idx} is outside the table's {vocab} rows")
        pad = padding_idx % vocab
    return torch.ops.gmdn.embed_fwd(weight, tokens, scale, pad)


class Embedding(nn.Embedding):
    """``nn.Embedding`` through ``embedding``, with a scale.  Its further options
    (``max_norm``, ``scale_grad_by_freq``, ``sparse``) are refused."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, scale: float = 1.0, **options):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, **options)
        for name in ("max_norm", "scale_grad_by_freq", "sparse"):
            if getattr(self, name):
                raise ValueError(f"{name} is not supported")
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings: Tensor, freeze: bool = True, padding_idx: int | None = None, scale: float = 1.0,
                        **options):
        """A module of this table; ``freeze``: without a gradient."""
        made = super().from_pretrained(embeddings, freeze=freeze, padding_idx=padding_idx, **options)
        made.scale = scale
        return made

    def forward(self, tokens: Tensor) -> Tensor:
        return embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, scale={self.scale}"
