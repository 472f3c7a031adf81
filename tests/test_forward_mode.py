"""Forward-mode derivatives: no operator has one, and an input that carries a
tangent is refused rather than returned without it, whether or not a gradient
is wanted.  On fake GPU tensors, so nothing runs on a device."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

from gmdn_amd import act8, layer_norm, logprobs
from gmdn_amd import ops  # noqa: F401
from test_ops import _meta_ops


def _lm_calls():
    """Name -> (call, its inputs), on the LM step's operators."""
    def t(*shape):
        return torch.empty(*shape, device="cuda")

    x, w, b, w1, w2 = t(4, 64), t(64), t(64), t(128, 64), t(64, 128)
    tokens = torch.empty(4, dtype=torch.int64, device="cuda")
    return {
        "layer_norm": (layer_norm.layer_norm, (x, w, b)),
        "layer_norm-int8": (lambda *a: layer_norm.layer_norm(*a, checkpoint="int8"), (x, w, b)),
        "gelu": (act8.gelu, (x,)),
        "mlp": (lambda *a: act8.mlp(*a, w2), (x, w1)),
        "norm_mlp": (lambda *a: act8.norm_mlp(*a, w2), (x, w, b, w1)),
        "token_logprobs": (lambda a: logprobs.token_logprobs(a, tokens, 2).logprob, (x,)),
        "cross_entropy": (lambda a: logprobs.cross_entropy(a, tokens), (x,)),
    }


def _refuses(call, inputs):
    """Each input in turn with a tangent, with and without a gradient wanted,
    and through torch.func.jvp."""
    for i, given in enumerate(inputs):
        def at(v, i=i):
            return call(*inputs[:i], v, *inputs[i + 1:])

        for grad in (False, True):
            with fwd.dual_level():
                dual = fwd.make_dual(given.clone().requires_grad_(grad), torch.empty_like(given))
                with pytest.raises(NotImplementedError, match="forward|jvp"):
                    at(dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward|jvp"):
                    at(dual)
        with pytest.raises(NotImplementedError, match="forward|jvp"):
            torch.func.jvp(at, (given,), (torch.empty_like(given),))
    call(*inputs)  # without tangents, also inside a level
    with fwd.dual_level():
        call(*inputs)


@pytest.mark.parametrize("name", ["layer_norm", "layer_norm-int8", "gelu", "mlp", "norm_mlp", "token_logprobs",
                                  "cross_entropy"])
def test_lm_operators_refuse_tangents(name):
    with FakeTensorMode():
        _refuses(*_lm_calls()[name])


def test_products_behind_them_keep_theirs():
    """A tangent that meets no operator of this package goes through: the
    second weight's, and linear's."""
    with FakeTensorMode(), fwd.dual_level():
        x, w1, w2 = (torch.empty(*s, device="cuda") for s in ((4, 64), (128, 64), (64, 128)))

        def dual(t):
            return fwd.make_dual(t, torch.empty_like(t))

        assert fwd.unpack_dual(act8.mlp(x, w1, dual(w2))).tangent is not None
        assert fwd.unpack_dual(act8.linear(dual(x), w1)).tangent is not None


@pytest.mark.parametrize("name", [x[0] for x in _meta_ops()])
def test_mixer_operators_refuse_tangents(name):
    _, call, inputs = next(x for x in _meta_ops() if x[0] == name)
    _refuses(call, [t.detach() for t in inputs])
