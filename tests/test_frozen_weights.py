"""The layers on 8-bit checkpoints with some of their inputs frozen: what the
forward keeps, and the gradients beside those with nothing frozen."""
import itertools

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from gmdn_amd import act8
from gmdn_amd import ops  # noqa: F401

D, HIDDEN, ROWS = 256, 640, 20
SHAPES = {"linear": [(ROWS, D), (HIDDEN, D), (HIDDEN,)],
          "mlp": [(ROWS, D), (HIDDEN, D), (D, HIDDEN)],
          "norm_mlp": [(ROWS, D), (D,), (D,), (HIDDEN, D), (D, HIDDEN)]}
# the inputs whose gradients read the input's checkpoint
READERS = {"linear": [1], "mlp": [1], "norm_mlp": [0, 1, 2, 3]}


def _kept(name, leaves):
    """Values kept in 8 bits by a call, by hooks on what it saves."""
    n = []

    def pack(t):
        if t.dtype == torch.int8:
            n.append(t.numel())
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        getattr(act8, name)(*leaves)
    return sum(n)


@pytest.mark.parametrize("name", list(SHAPES))
def test_no_checkpoint_for_frozen_weights(name):
    """An input's checkpoint is kept where a gradient reads it, and only there."""
    hidden = 0 if name == "linear" else ROWS * HIDDEN
    with FakeTensorMode():
        for wants in itertools.product((False, True), repeat=len(SHAPES[name])):
            if any(wants):
                leaves = [torch.empty(s, device="cuda", requires_grad=w) for s, w in zip(SHAPES[name], wants)]
                own = ROWS * D if any(wants[i] for i in READERS[name]) else 0
                assert _kept(name, leaves) == own + hidden, wants


@pytest.mark.parametrize("name", list(SHAPES))
def test_compiles_with_frozen_inputs(name):
    """Each layer in one graph, with the first weight frozen and with the input."""
    with FakeTensorMode():
        for frozen in (READERS[name][-1], 0, None):
            leaves = [torch.empty(s, device="cuda", requires_grad=i != frozen) for i, s in enumerate(SHAPES[name])]
            torch._dynamo.reset()
            out = torch.compile(getattr(act8, name), backend="eager", fullgraph=True)(*leaves)
            assert out.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("name", list(SHAPES))
def test_gradients_with_frozen_inputs(name, autocast):
    """Whatever is frozen, the other gradients are those with nothing frozen,
    bit for bit: the same kernels on the same values."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    gen = torch.Generator().manual_seed(3)
    values = [torch.randn(s, generator=gen).cuda() / s[-1] ** 0.5 for s in SHAPES[name]]
    dy = None

    def grads(wants):
        nonlocal dy
        leaves = [v.clone().requires_grad_(w) for v, w in zip(values, wants)]
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            out = getattr(act8, name)(*leaves)
        if dy is None:
            dy = torch.randn(out.shape, generator=gen).to(out)
        out.backward(dy)
        assert all((t.grad is not None) == w for t, w in zip(leaves, wants))
        return [t.grad for t in leaves]

    whole = grads([True] * len(values))
    for wants in itertools.product((False, True), repeat=len(values)):
        if any(wants):
            for g, ref in zip(grads(wants), whole):
                assert g is None or torch.equal(g, ref), wants
