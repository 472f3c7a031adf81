"""The residual stream's operators in the LM: run together, beside torch's own
modules, captured and replayed, on another stream."""
import pytest
import torch
import torch.nn as nn

from gmdn_amd import embedding, logprobs, residual
from gmdn_amd import ops  # noqa: F401
from gmdn_amd.mixer import LM, Branch

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _pair(dev, dtype, **kw):
    """An LM on the operators and the same one on torch's modules."""
    torch.manual_seed(0)
    ours = LM(300, 128, 2, 2, "delta", residual="fused", loss="linear", embedding="sorted", **kw)
    theirs = LM(300, 128, 2, 2, "delta")
    theirs.load_state_dict(ours.state_dict())
    return ours.to(dev, dtype), theirs.to(dev, dtype)


def _step(model, idx, autocast):
    with torch.autocast(idx.device.type, dtype=torch.bfloat16, enabled=autocast):
        _, loss = model(idx[:, :-1], idx[:, 1:])
    model.zero_grad(set_to_none=True)
    loss.backward()
    return loss.detach(), {n: p.grad for n, p in model.named_parameters()}


@pytest.mark.parametrize("dtype,autocast", [(torch.float32, False), (torch.float32, True), (torch.bfloat16, False)])
def test_step_beside_torch_modules(dtype, autocast):
    """Loss and gradients of one step.  In float32 the two differ by the order of
    their sums and the head's split products; in bfloat16 each rounds the stream, the
    norms and the logits in other places, so they are compared by their direction."""
    dev = _dev()
    ours, theirs = _pair(dev, dtype)
    idx = torch.randint(300, (2, 129), generator=torch.Generator().manual_seed(1)).to(dev)
    (la, ga), (lb, gb) = _step(ours, idx, autocast), _step(theirs, idx, autocast)
    assert set(ga) == set(gb)
    exact = dtype == torch.float32 and not autocast
    assert abs(float(la) - float(lb)) < (1e-4 if exact else 0.05) * float(lb)
    for n, g in ga.items():
        a, b = g.double().flatten(), gb[n].double().flatten()
        assert a.isfinite().all() and g.dtype == gb[n].dtype
        cos = float(a @ b / (a.norm() * b.norm()).clamp_min(1e-300))
        assert cos > (1 - 1e-5 if exact else 0.97), (n, cos)


def test_scoring_beside_the_logits():
    dev = _dev()
    ours, _ = _pair(dev, torch.float32)
    idx = torch.randint(300, (2, 128), generator=torch.Generator().manual_seed(2)).to(dev)
    a, b = ours.score(idx), logprobs.token_logprobs(ours(idx)[0].detach(),
                                                    nn.functional.pad(idx[:, 1:], (0, 1), value=logprobs.IGNORE))
    assert a.top_tokens.shape == (2, 128, 0)
    # three bfloat16 pieces' products beside float32 sums of 128 terms below 1
    assert (a.logprob - b.logprob).abs().max() < 1e-3 and (a.entropy - b.entropy).abs().max() < 1e-3
    assert (a.logprob[:, -1] == 0).all()


def test_all_options_train():
    """Post norms, gates and scales in a step under autocast: every parameter has
    a gradient, and the one of a scale is a difference's."""
    dev = _dev()
    torch.manual_seed(0)
    model = LM(300, 128, 2, 2, "delta", residual="fused", loss="linear", embedding="sorted", emb_scale=11.0, post_norm=True,
               gated=True, layer_scale=0.5).to(dev)
    idx = torch.randint(300, (2, 129), generator=torch.Generator().manual_seed(3)).to(dev)
    _, grads = _step(model, idx, True)
    assert all(g is not None and g.isfinite().all() and g.abs().max() > 0 for g in grads.values())
    _, grads = _step(model, idx, False)
    p = model.blocks[1].join2.scale
    direction = torch.sign(grads["blocks.1.join2.scale"])
    h, losses = 2.0 ** -6, []
    for sign in (1, -1):
        with torch.no_grad():
            p.add_(sign * h * direction)
            losses.append(float(model(idx[:, :-1], idx[:, 1:])[1]))
            p.sub_(sign * h * direction)
    slope = float((grads["blocks.1.join2.scale"] * direction).sum())
    assert abs((losses[0] - losses[1]) / (2 * h) - slope) < 0.05 * slope + 2e-3


def test_branch_beside_modules():
    """A branch's parts inside the operator beside the same by torch."""
    dev = _dev()
    gen = torch.Generator().manual_seed(4)
    torch.manual_seed(4)
    branch, norm = Branch(96, True, True, 0.3).to(dev), nn.RMSNorm(96).to(dev)
    x, y, z = (torch.randn(3, 7, 96, generator=gen).to(dev).requires_grad_(True) for _ in range(3))
    r, out = branch(x, y, z, norm)
    want = x + branch.scale * torch.sigmoid(branch.gate(z)) * branch.post(y)
    cot = [torch.randn(3, 7, 96, generator=gen).to(dev) for _ in range(2)]
    leaves = [x, y, z, *branch.parameters(), *norm.parameters()]
    a = torch.autograd.grad([r, out], leaves, cot)
    b = torch.autograd.grad([want, norm(want)], leaves, cot)
    for g, ref in zip((r, out, *a), (want, norm(want), *b)):
        assert torch.allclose(g, ref, rtol=1e-4, atol=1e-4)


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


@pytest.mark.parametrize("rows,vocab", [(300, 9001), (3, 700)])
def test_replays(rows, vocab):
    """Lookup, residuals and loss with their gradients in one graph: every replay
    is the eager step on the inputs of the moment."""
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(5)
    D = 136

    def t(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    table, w, scale, y, gate = (v.requires_grad_(True) for v in (t(vocab, D), t(D), t(D), t(rows, D), t(rows, D)))
    tokens = torch.randint(vocab, (rows,), generator=gen, device=dev)
    targets = torch.randint(vocab, (rows,), generator=gen, device=dev)
    leaves = [table, w, scale, y, gate]

    def step():
        x = embedding.embedding(tokens, table, 3.0)
        x, z = residual.residual_norm(x, y, w, post_weight=scale, gate=gate, scale=scale)
        x, z = residual.residual_norm(x, z, w)
        lp, h = logprobs.linear_logprobs(z, table, targets)
        return (lp, h, *torch.autograd.grad([lp, h, x], leaves, [torch.ones_like(lp), torch.ones_like(h), y.detach()]))

    graph, outs = _capture(step)
    before = None
    for rep in range(4):
        with torch.no_grad():
            for v in leaves:
                v.normal_(generator=gen).mul_(0.1 + 0.05 * rep)
            for v in (tokens, targets):
                v.copy_(torch.randint(vocab, (rows,), generator=gen, device=dev))
        want = [v.detach().clone() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), f"replay {rep}: output {k} differs"
        assert before is None or not any(torch.equal(a, b) for a, b in zip(outs, before)), "inputs did not change"
        before = [v.detach().clone() for v in outs]


def test_two_streams_at_once():
    """Two calls on streams of their own, with workspaces of their own: each is
    what it is alone."""
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(6)
    sets = [(torch.randn(500, 64, generator=gen, device=dev), torch.randn(3001, 64, generator=gen, device=dev),
             torch.randint(3001, (500,), generator=gen, device=dev)) for _ in range(2)]

    def call(x, w, tokens):
        lp, h, stats = torch.ops.gmdn.linear_logprobs_fwd(x, w, tokens, -100)
        dx, dw = torch.ops.gmdn.linear_logprobs_bwd(x, w, tokens, stats, h, lp, None, -100, True, True)
        return lp, dx, dw, torch.ops.gmdn.embed_bwd(x, tokens, 3001, 1.0, -1)

    alone = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(call(*s))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
