"""An LM calls the modules that a user has put in a block's place (fake tensors: no
kernel runs)."""
import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

from gmdn_amd import ops  # noqa: F401
from gmdn_amd.mixer import LM
from test_stream_ops_cpu import _ops_of

def _lm(**kw):
    lm = LM(50, 64, 3, 2, "delta", **kw)
    for blk in lm.blocks:
        blk.mixer = nn.Linear(64, 64)
    return lm


@pytest.mark.parametrize("kw", [{}, {"residual": "fused"}])
def test_replaced_blocks(kw):
    with FakeTensorMode(), torch.device("cuda"):
        idx = torch.empty(2, 64, dtype=torch.int64)
        lm = _lm(**kw)
        lm.blocks[1] = nn.Identity()
        assert lm(idx)[0].shape == (2, 64, 50)
        assert _ops_of(lambda: lm(idx)) == (["residual_norm_fwd"] * 2 if kw else [])
