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


def _linear_branches(model):
    """A linear layer in place of each block's mixer.  Chains of chunk updates near
    their initialisation turn a last bit of their input into another gradient
    altogether, so that nothing could be compared behind them."""
    for blk in model.blocks:
        blk.mixer = nn.Linear(128, 128, bias=False)
        nn.init.normal_(blk.mixer.weight, std=0.05)
    return model


def _pair(dev, dtype):
    """An LM on the operators and the same one on torch's modules."""
    torch.manual_seed(0)
    ours = _linear_branches(LM(300, 128, 2, 2, "delta", residual="fused", loss="linear", embedding="sorted"))
    theirs = _linear_branches(LM(300, 128, 2, 2, "delta"))
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
    their sums (some hundred terms: 2^-16 of a value) and the head's split products (3
    2^-16): below 1e-3 after two blocks.  Around bfloat16 products and streams each rounds
    values at other places, 2^-8 each; some ten of them that add up at random turn a gradient
    by 2^-8 sqrt(10), and 0.15 allows for twelve times that."""
    dev = _dev()
    ours, theirs = _pair(dev, dtype)
    idx = torch.randint(300, (2, 129), generator=torch.Generator().manual_seed(1)).to(dev)
    (la, ga), (lb, gb) = _step(ours, idx, autocast), _step(theirs, idx, autocast)
    assert set(ga) == set(gb)
    tol = 1e-3 if dtype == torch.float32 and not autocast else 0.15
    assert abs(float(la) - float(lb)) < tol * float(lb)
    for n, g in ga.items():
        a, b = g.double().flatten(), gb[n].double().flatten()
        assert a.isfinite().all() and g.dtype == gb[n].dtype
        assert float((a - b).norm()) < tol * float(b.norm()), (n, float((a - b).norm() / b.norm()))


def test_scoring_beside_the_logits():
    dev = _dev()
    ours, _ = _pair(dev, torch.float32)
    idx = torch.randint(300, (2, 128), generator=torch.Generator().manual_seed(2)).to(dev)
    a, b = ours.score(idx), logprobs.token_logprobs(ours(idx)[0].detach(),
                                                    nn.functional.pad(idx[:, 1:], (0, 1), value=logprobs.IGNORE))
    assert a.top_tokens.shape == (2, 128, 0)
    # split products beside float32 sums of 128 terms below 1
    assert (a.logprob - b.logprob).abs().max() < 1e-3 and (a.entropy - b.entropy).abs().max() < 1e-3
    assert (a.logprob[:, -1] == 0).all()


@pytest.mark.parametrize("inner", ["delta", "muon"])
def test_step_around_the_mixer(inner):
    """All options around the mixer's own kernels, under autocast: every parameter
    has a gradient.  (A gate's bias before a sigmoid's logarithm may have none
    of size.)"""
    dev = _dev()
    torch.manual_seed(0)
    model = LM(300, 128, 2, 2, inner, residual="fused", loss="linear", embedding="sorted", emb_scale=11.0, post_norm=True,
               gated=True, layer_scale=0.5).to(dev)
    idx = torch.randint(300, (2, 129), generator=torch.Generator().manual_seed(3)).to(dev)
    loss, grads = _step(model, idx, True)
    assert 0 < float(loss) < 20
    assert all(g is not None and g.isfinite().all() for g in grads.values())
    for n in ("emb.weight", "norm_f.weight", "blocks.0.join1.post.weight", "blocks.0.join1.gate.weight",
              "blocks.0.join1.scale", "blocks.1.join2.scale", "blocks.1.mlp.2.weight"):
        assert grads[n].abs().max() > 0, n


def test_kept_activations_in_8_bits():
    """checkpoint="int8" in blocks whose norm comes from the residual's pass."""
    dev = _dev()
    torch.manual_seed(0)
    kw = dict(residual="fused", loss="linear", embedding="sorted")
    plain, kept = (_linear_branches(LM(300, 128, 2, 2, "delta", checkpoint=c, **kw)) for c in (None, "int8"))
    kept.load_state_dict(plain.state_dict())
    plain, kept = plain.to(dev), kept.to(dev)
    idx = torch.randint(300, (2, 129), generator=torch.Generator().manual_seed(4)).to(dev)
    (la, ga), (lb, gb) = _step(kept, idx, False), _step(plain, idx, False)
    assert abs(float(la) - float(lb)) < 1e-4 * float(lb)
    for n, g in ga.items():  # activations within 1 / 254 of their group's largest
        assert float((g - gb[n]).norm()) < 0.1 * float(gb[n].norm()), n


def test_slope_of_a_scale():
    """A layer scale's gradient beside differences of the whole loss."""
    dev = _dev()
    torch.manual_seed(0)
    model = _linear_branches(LM(300, 128, 2, 2, "delta", residual="fused", loss="linear", embedding="sorted", emb_scale=11.0,
                                post_norm=True, gated=True, layer_scale=0.5)).to(dev)
    idx = torch.randint(300, (2, 129), generator=torch.Generator().manual_seed(3)).to(dev)
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
    # h^2 / 6 of a third derivative, and the loss's rounding (2^-21) over 2 h
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


def _op_calls(dev):
    """Name -> arguments of every operator, by the shapes of one another's results."""
    gen = torch.Generator().manual_seed(7)

    def t(*shape):
        return torch.randn(*shape, generator=gen).to(dev)

    op = torch.ops.gmdn
    w, x, v = t(50, 24), t(2, 5, 24), t(24)
    tokens = torch.randint(50, (2, 5), generator=gen).to(dev)
    r, z, rstd, post = op.residual_norm_fwd(x, x, v, v, x, v, 1e-6)
    lp, h, stats = op.linear_logprobs_fwd(x, w, tokens, -100)

    def leaf(u):
        return u.clone().requires_grad_(True)

    return {"embed_fwd": (leaf(w), tokens, 2.0, 3), "embed_bwd": (x, tokens, 50, 2.0, -1),
            "residual_norm_fwd": (leaf(x), leaf(x), leaf(v), leaf(v), leaf(x), leaf(v), 1e-6),
            "residual_norm_bwd": (x, None, r, x, v, v, x, v, rstd, post),
            "linear_logprobs_fwd": (leaf(x), leaf(w), tokens, -100),
            "linear_logprobs_bwd": (x, w, tokens, stats, h, h, None, -100, True, True)}


@pytest.mark.parametrize("name", ["embed_fwd", "embed_bwd", "residual_norm_fwd", "residual_norm_bwd",
                                  "linear_logprobs_fwd", "linear_logprobs_bwd"])
def test_opcheck(name):
    dev = _dev()
    torch.library.opcheck(getattr(torch.ops.gmdn, name).default, _op_calls(dev)[name])
