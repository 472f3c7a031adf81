"""The LM step's operators in a HIP graph with inputs that change in place
between its replays: every replay is the eager step on the inputs of the
moment."""
import pytest
import torch

from gmdn_amd import act8, layer_norm, logprobs
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
ROWS, D, V = 300, 256, 9001


def _capture(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    torch.cuda.synchronize()
    return graph, outs


def _replays(step, refill):
    graph, outs = _capture(step)
    before = None
    for rep in range(4):
        with torch.no_grad():
            refill(rep)
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), f"replay {rep}: output {k} differs"
        assert before is None or not any(torch.equal(a, b) for a, b in zip(outs, before)), "inputs did not change"
        before = [t.detach().clone() for t in outs]


def test_norm_and_mlp():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    gen = torch.Generator(device="cuda").manual_seed(0)

    def t(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    leaves = [t(ROWS, D), t(D), t(D), t(4 * D, D) / 16, t(D, 4 * D) / 32]
    dy = t(ROWS, D)
    leaves = [v.requires_grad_(True) for v in leaves]

    def step():
        y = act8.norm_mlp(*leaves)
        z = layer_norm.layer_norm(y, *leaves[1:3], checkpoint="int8")
        return (y, z, *torch.autograd.grad(z, leaves, dy))

    def refill(rep):
        for v in (*leaves, dy):
            v.normal_(generator=gen).mul_(0.1 + 0.1 * rep)

    _replays(step, refill)


@pytest.mark.parametrize("rows,top", [(ROWS, 0), (ROWS, 5), (2, 0)])
def test_log_probabilities(rows, top):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = V if rows > 2 else 90001
    x = torch.randn(rows, wide, generator=gen, device="cuda").requires_grad_(True)
    tokens = torch.randint(wide, (rows,), generator=gen, device="cuda")
    g = torch.randn(rows, generator=gen, device="cuda")

    def step():
        got = logprobs.token_logprobs(x, tokens, top)
        (d,) = torch.autograd.grad(got[:2], x, [g, g])
        return got.logprob, got.entropy, *(got[2:] if top else ()), d

    def refill(rep):
        x.normal_(generator=gen).mul_(2.0 + rep)
        tokens.copy_(torch.randint(wide, (rows,), generator=gen, device="cuda"))
        g.normal_(generator=gen)

    _replays(step, refill)
