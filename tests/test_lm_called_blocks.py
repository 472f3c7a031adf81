"""An LM of fused residuals calls the modules that a user has put in a block's place,
compiled in place or watches by hooks of all modules, and goes from block to block by
itself only where nobody would notice (fake tensors: no kernel runs)."""
import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

from gmdn_amd import ops  # noqa: F401
from gmdn_amd.mixer import LM, Block
from test_stream_ops_cpu import _ops_of

ACROSS = ["residual_norm_fwd"] * 6  # three blocks in one chain
WITHIN = ["residual_norm_fwd"] * 3


def _lm(**kw):
    lm = LM(50, 64, 3, 2, "delta", **kw)
    for blk in lm.blocks:
        blk.mixer = nn.Linear(64, 64)
    return lm


@pytest.mark.parametrize("at", [0, 1])
@pytest.mark.parametrize("kw", [{}, {"residual": "fused"}])
def test_replaced_blocks(kw, at):
    with FakeTensorMode(), torch.device("cuda"):
        idx = torch.empty(2, 64, dtype=torch.int64)
        lm = _lm(**kw)
        lm.blocks[at] = nn.Identity()
        assert lm(idx)[0].shape == (2, 64, 50)
        assert _ops_of(lambda: lm(idx)) == (["residual_norm_fwd"] * 2 if kw else [])


def test_compiled_blocks():
    torch._dynamo.reset()
    with FakeTensorMode(), torch.device("cuda"):
        idx = torch.empty(2, 64, dtype=torch.int64)
        lm = _lm(residual="fused")
        assert _ops_of(lambda: lm(idx)) == ACROSS
        ran = []

        def backend(gm, inputs):
            return lambda *a: ran.append(1) or gm(*a)

        lm.blocks[1].compile(backend=backend)
        lm(idx)
        assert ran


def test_compiled_norms():
    """(torch.compile leaves a lone torch.nn module's call as it is, so the call itself is watched.)"""
    torch._dynamo.reset()
    with FakeTensorMode(), torch.device("cuda"):
        lm, ran = _lm(residual="fused"), []
        norm = lm.blocks[1].n2
        norm.compile(backend="eager")
        compiled = norm._compiled_call_impl
        norm._compiled_call_impl = lambda *a: ran.append(1) or compiled(*a)
        lm(torch.empty(2, 64, dtype=torch.int64))
        assert ran == [1]


def test_hooks_of_all_modules():
    with FakeTensorMode(), torch.device("cuda"):
        idx = torch.empty(2, 64, dtype=torch.int64)
        lm, seen = _lm(residual="fused"), []
        handle = nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(type(m)))
        try:
            assert _ops_of(lambda: lm(idx)) == WITHIN
        finally:
            handle.remove()
        assert seen.count(Block) == 3 and seen.count(nn.RMSNorm) == 7 and seen.count(nn.GELU) == 3
        assert _ops_of(lambda: lm(idx)) == ACROSS
