"""The block's 8-bit MLP beside modules that are not the plain ones any more:
hooks are called, and a replaced module, a bias or another activation counts."""
import copy

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from gmdn_amd import ops  # noqa: F401
from gmdn_amd.mixer import Block

D = 64


class _Ops(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.add(str(func))
        return func(*args, **(kwargs or {}))


def _kept8(block, x):
    """(MLP's hidden layer in 8 bits, the norm's input in 8 bits) of a call."""
    with _Ops() as seen:
        block._mlp(x)
    return "gmdn.gelu8_fwd.default" in seen.names, "gmdn.layer_norm_fwd.default" in seen.names


class _Adapter(nn.Linear):
    def __init__(self, base):
        super().__init__(base.in_features, base.out_features, bias=False)
        self.weight = base.weight
        self.up, self.down = nn.Parameter(torch.ones(base.out_features, 2)), nn.Parameter(torch.ones(2, base.in_features))

    def forward(self, x):
        return super().forward(x) + x @ self.down.t() @ self.up.t()


def _replace(what, block):
    """Changes the block's MLP or norm as users do."""
    m = block.mlp
    if what == "adapter":
        m[0] = _Adapter(m[0])
    elif what == "bias":
        m[2] = nn.Linear(4 * D, D)
    elif what == "activation":
        m[1] = nn.SiLU()
    elif what == "tanh":
        m[1] = nn.GELU(approximate="tanh")
    elif what == "dropout":
        m.append(nn.Dropout(0.5))
    elif what == "forward":
        plain = m[0].forward
        m[0].forward = lambda x: 2 * plain(x)
    elif what == "sequential":
        block.mlp = nn.Sequential(*m, nn.Tanh())


CHANGES = ["adapter", "bias", "activation", "tanh", "dropout", "forward", "sequential"]


FORWARD = ["register_forward_hook", "register_forward_pre_hook"]
BACKWARD = ["register_full_backward_hook", "register_full_backward_pre_hook"]


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("place", ["mlp", "mlp.0", "mlp.1", "mlp.2"])
@pytest.mark.parametrize("hook", FORWARD + BACKWARD)
def test_hooked_modules_are_called(hook, place, norm):
    with FakeTensorMode(), torch.device("cuda"):
        block, x, seen = Block(D, 2, "delta", 64, norm=norm, checkpoint="int8"), torch.empty(3, 5, D, requires_grad=True), []
        assert _kept8(block, x)[0]
        handle = getattr(block.get_submodule(place), hook)(lambda *a: seen.append(place))
        assert not _kept8(block, x)[0]
        assert seen == ([place] if hook in FORWARD else [])
        handle.remove()
        assert _kept8(block, x)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("hook", FORWARD + BACKWARD)
def test_hooks_see_a_step(hook):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    block, seen = Block(D, 2, "delta", 64, norm="layer", checkpoint="int8").cuda(), []
    for place in ("n2", "mlp", "mlp.0", "mlp.1", "mlp.2"):
        getattr(block.get_submodule(place), hook)(lambda *a, place=place: seen.append(place))
    block._mlp(torch.randn(3, 64, D, device="cuda", requires_grad=True)).sum().backward()
    assert sorted(seen) == ["mlp", "mlp.0", "mlp.1", "mlp.2", "n2"]


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_hooks_of_the_norm_are_called(norm):
    """The MLP keeps its own checkpoints beside a norm that is called."""
    with FakeTensorMode(), torch.device("cuda"):
        block, x, seen = Block(D, 2, "delta", 64, norm=norm, checkpoint="int8"), torch.empty(3, 5, D, requires_grad=True), []
        block.n2.register_forward_hook(lambda *a: seen.append("n2"))
        assert _kept8(block, x) == (True, norm == "layer") and seen == ["n2"]


@pytest.mark.parametrize("what", CHANGES)
def test_replaced_modules_are_called(what):
    with FakeTensorMode(), torch.device("cuda"):
        block, x = Block(D, 2, "delta", 64, norm="layer", checkpoint="int8"), torch.empty(3, 5, D, requires_grad=True)
        _replace(what, block)
        assert _kept8(block, x) == (False, True)


def test_parametrized_weights_keep_their_checkpoints():
    """A weight computed by a parametrization is the module's weight still."""
    class Double(nn.Module):
        def forward(self, w):
            return 2 * w

    with FakeTensorMode(), torch.device("cuda"):
        block, x = Block(D, 2, "delta", 64, norm="layer", checkpoint="int8"), torch.empty(3, 5, D, requires_grad=True)
        nn.utils.parametrize.register_parametrization(block.mlp[0], "weight", Double())
        assert _kept8(block, x)[0]


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_compiles_to_one_graph(norm):
    with FakeTensorMode(), torch.device("cuda"):
        block, x = Block(D, 2, "delta", 64, norm=norm, checkpoint="int8"), torch.empty(3, 5, D, requires_grad=True)
        torch._dynamo.reset()
        assert torch.compile(block._mlp, backend="eager", fullgraph=True)(x).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("what", CHANGES)
def test_replaced_modules_give_what_they_give_without_checkpoints(what):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(0)
    block = Block(D, 2, "delta", 64, norm="rms", checkpoint="int8").cuda()
    _replace(what, block)
    block.cuda().eval()  # (the dropout)
    plain = copy.deepcopy(block)
    plain.keep8 = False
    x = torch.randn(3, 64, D, device="cuda")
    assert torch.equal(block._mlp(x), plain._mlp(x))
