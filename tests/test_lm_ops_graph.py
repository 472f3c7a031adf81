"""The LM step's operators, forward and backward, traced into one graph: what
torch.compile's partitioner sees.  On meta tensors, so nothing runs on a
device."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from gmdn_amd import act8, layer_norm, logprobs
from gmdn_amd import ops  # noqa: F401


def _calls():
    def t(*shape):
        return torch.empty(*shape, device="meta")

    x, w, b, w1 = t(4, 64), t(64), t(64), t(128, 64)
    norm, norm8 = ["layer_norm_fwd", "layer_norm_bwd"], ["layer_norm_fwd", "layer_norm8_bwd"]
    return {
        "norm": (lambda t, *a: layer_norm.layer_norm(*a), (x, w, b), norm),
        "norm-int8": (lambda t, *a: layer_norm.layer_norm(*a, checkpoint="int8"), (x, w, b), norm8),
        "gelu": (lambda t, a: act8.gelu(a), (x,), ["gelu8_fwd", "gelu8_bwd"]),
        "lp": (lambda t, a: sum(v.sum() for v in logprobs.token_logprobs(a, t, 3)[:3]), (x,),
               ["logprobs_fwd", "logprobs_bwd"]),
        "loss": (lambda t, a: logprobs.cross_entropy(a, t), (x,), ["logprobs_fwd", "logprobs_bwd"]),
        "step": (lambda t, x, w, b, h: logprobs.cross_entropy(act8.gelu(layer_norm.layer_norm(x, w, b) @ h.t()), t),
                 (x, w, b, w1), norm + ["gelu8_fwd", "gelu8_bwd", "logprobs_fwd", "logprobs_bwd"]),
    }


@pytest.mark.parametrize("name", ["norm", "norm-int8", "gelu", "lp", "loss", "step"])
def test_forward_and_backward_trace_to_one_graph(name):
    call, inputs, wanted = _calls()[name]

    def step(tokens, *xs):
        xs = [x.detach().requires_grad_() for x in xs]
        out = call(tokens, *xs)
        return torch.autograd.grad(out, xs, torch.empty_like(out))

    gm = make_fx(step, tracing_mode="symbolic")(torch.empty(4, dtype=torch.int64, device="meta"), *inputs)
    seen = [str(n.target).split(".")[1] for n in gm.graph.nodes if "gmdn" in str(n.target)]
    assert sorted(seen) == sorted(wanted)
    grads = next(n for n in gm.graph.nodes if n.op == "output").args[0]
    assert [g.meta["val"].shape for g in grads] == [x.shape for x in inputs]
