"""The LM stack with layer norm, 8-bit activation checkpoints and the loss from
the log probabilities: against the same stack with torch's modules, its
scoring, and the step under HIP graph capture."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from gmdn_amd import act8, layer_norm, logprobs
from gmdn_amd.mixer import LM

pytestmark = pytest.mark.gpu
VOCAB = 1000


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _model(dev, norm, checkpoint=None, loss="torch", dtype=None):
    torch.manual_seed(0)
    model = LM(VOCAB, 256, 2, 2, "delta", norm=norm, checkpoint=checkpoint, loss=loss).to(dev)
    return model.to(dtype) if dtype else model


def _step(model, idx, autocast):
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        logits, loss = model(idx[:, :-1], idx[:, 1:])
    return logits, loss, dict(zip([n for n, _ in model.named_parameters()],
                                  torch.autograd.grad(loss, list(model.parameters()))))


def _moved(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def _batch(dev):
    gen = torch.Generator().manual_seed(1)
    return torch.randint(VOCAB, (2, 257), generator=gen).to(dev)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("mode", ["f32", "autocast", "bf16"])
def test_lm_step_beside_torch(norm, mode, monkeypatch):
    """The same parameters with every option and with none (layer norms by
    torch there).  The loss is the same up to the type's rounding; gradients
    move by what 8 bits in two places a block and the type may: 2 % each,
    four times (as for one MLP, twice as deep), 2^-8 a value for bfloat16."""
    dev = _dev()
    dtype = torch.bfloat16 if mode == "bf16" else None
    mine = _model(dev, norm, "int8", "logprobs", dtype)
    plain = _model(dev, norm, None, "torch", dtype)
    plain.load_state_dict(mine.state_dict())
    for m in plain.modules():
        if isinstance(m, layer_norm.LayerNorm):
            monkeypatch.setattr(m, "forward", lambda x, m=m: nn.LayerNorm.forward(m, x))
    idx = _batch(dev)
    _, loss, grads = _step(mine, idx, mode == "autocast")
    _, ref, want = _step(plain, idx, mode == "autocast")
    assert loss.dtype == torch.float32
    assert abs(loss.item() - ref.item()) <= (1e-5 if mode == "f32" else 0.02) * ref.item()
    for name, g in grads.items():
        assert torch.isfinite(g).all() and g.dtype == want[name].dtype, name
        if mode == "f32":
            assert _moved(g, want[name]) < 0.08, name
    whole = torch.cat([g.double().flatten() for g in grads.values()])
    other = torch.cat([want[n].double().flatten() for n in grads])
    assert _moved(whole, other) < (0.04 if mode == "f32" else 0.08)


def test_default_lm_takes_none_of_it(monkeypatch):
    """Without options the stack runs torch's norms, MLP and loss as before."""
    dev = _dev()
    for mod, name in ((act8, "mlp"), (act8, "norm_mlp"), (logprobs, "cross_entropy"), (layer_norm, "layer_norm")):
        monkeypatch.setattr(mod, name, lambda *a, **k: pytest.fail("not the default's path"))
    logits, loss, _ = _step(_model(dev, "rms", dtype=torch.bfloat16), _batch(dev), False)
    ref = F.cross_entropy(logits.view(-1, VOCAB).float(), _batch(dev)[:, 1:].reshape(-1))
    assert torch.equal(loss, ref)


def test_score():
    """Scores of a prompt: each next token's log probability, entropies and
    alternatives, beside torch's log softmax of the logits."""
    dev = _dev()
    model, idx = _model(dev, "layer", dtype=torch.bfloat16), _batch(dev)[:, :256]
    got = model.score(idx, top=5)
    with torch.no_grad():
        logits = model(idx)[0]
    ref = torch.log_softmax(logits.double(), -1)
    want = ref[:, :-1].gather(-1, idx[:, 1:, None])[..., 0]
    assert got.logprob.shape == idx.shape and got.logprob[:, -1].eq(0).all()
    assert (got.logprob[:, :-1] - want).abs().max() < 1e-5
    assert (got.entropy + (ref.exp() * ref).sum(-1)).abs().max() < 1e-5
    order = torch.argsort(logits.float(), dim=-1, descending=True, stable=True)[..., :5]
    assert torch.equal(got.top_tokens, order)
    some = torch.randint(VOCAB, idx.shape, device=dev)
    assert (model.score(idx, some).logprob - ref.gather(-1, some[..., None])[..., 0]).abs().max() < 1e-5


def test_graph_replays_match_eager():
    """Forward and backward of all of it captured in one HIP graph: each replay
    gives the eager step's bits, with eager work and synchronisations between."""
    dev = _dev()
    torch.manual_seed(0)
    x = torch.randn(300, 256, device=dev, requires_grad=True)
    nw = torch.rand(256, device=dev).requires_grad_(True)
    nb = torch.zeros(256, device=dev).requires_grad_(True)
    w1 = (torch.randn(1024, 256, device=dev) / 16).requires_grad_(True)
    w2 = (torch.randn(256, 1024, device=dev) / 32).requires_grad_(True)
    dy = torch.randn(300, 256, device=dev)
    tokens = torch.randint(256, (300,), device=dev)
    leaves = (x, nw, nb, w1, w2)

    def step():
        y = act8.norm_mlp(x, nw, nb, w1, w2)
        z = layer_norm.layer_norm(y, nw, nb, checkpoint="int8")
        got = logprobs.token_logprobs(z, tokens, 3)
        return (y, z, *got, *torch.autograd.grad((z, got.logprob, got.entropy), leaves,
                                                 (dy, dy[:, 0].contiguous(), dy[:, 1].contiguous())))

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
    ref = [t.detach().clone() for t in step()]
    for rep in range(3):
        step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(outs, ref)):
            assert torch.equal(a, b), f"replay {rep}: output {k} differs"


def test_loss_graph_replays_match_eager():
    """The mean loss over many tokens, forward and backward, in one graph."""
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(20000, 96, generator=gen, device=dev, dtype=torch.bfloat16).requires_grad_(True)
    targets = torch.randint(96, (20000,), generator=gen, device=dev)
    targets[::17] = logprobs.IGNORE

    def step():
        loss = logprobs.cross_entropy(x, targets)
        return loss, *torch.autograd.grad(loss, x)

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
    ref = [t.detach().clone() for t in step()]
    for rep in range(4):
        step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(outs, ref)):
            assert torch.equal(a, b), f"replay {rep}: output {k} differs"


def _op_calls(dev):
    gen = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(6, 5, 200, generator=gen, device=dev).requires_grad_(True)
    w, b = (torch.randn(200, generator=gen, device=dev).requires_grad_(True) for _ in range(2))
    tokens = torch.randint(200, (6, 5), generator=gen, device=dev)
    plain = x.detach()
    with torch.no_grad():
        y, mean, rstd, q, scale = torch.ops.gmdn.layer_norm_fwd(plain, w, b, 1e-5, torch.float32, True)
        _, h, _, top, stats = torch.ops.gmdn.logprobs_fwd(plain, tokens, 3, -100)
    wd, bd = w.detach(), b.detach()
    return {
        "layer_norm_fwd": (x, w, b, 1e-5, torch.bfloat16, False),
        "layer_norm_bwd": (y, plain, wd, mean, rstd),
        "layer_norm8_bwd": (y, q, scale, wd, mean, rstd, torch.float32),
        "layer_norm8_rebuild": (q, scale, wd, bd, mean, rstd, torch.bfloat16),
        "act8_pack": (plain,),
        "act8_unpack": (q, scale, torch.bfloat16),
        "gelu8_fwd": (x,),
        "gelu8_bwd": (y, q, scale, True),
        "logprobs_fwd": (x, tokens, 3, -100),
        "logprobs_bwd": (plain, tokens, stats, h, top, h, None, None, -100),
    }


@pytest.mark.parametrize("name", ["layer_norm_fwd", "layer_norm_bwd", "layer_norm8_bwd", "layer_norm8_rebuild",
                                  "act8_pack", "act8_unpack", "gelu8_fwd", "gelu8_bwd", "logprobs_fwd", "logprobs_bwd"])
def test_opcheck(name):
    dev = _dev()
    torch.library.opcheck(getattr(torch.ops.gmdn, name).default, _op_calls(dev)[name])


def test_compiled_step_matches_eager():
    """torch.compile over norm, MLP and loss with 8-bit checkpoints: the eager
    call's loss and gradients."""
    dev = _dev()
    torch.manual_seed(0)
    x = torch.randn(4, 60, 64, device=dev, requires_grad=True)
    nw, nb = torch.rand(64, device=dev).requires_grad_(True), torch.zeros(64, device=dev, requires_grad=True)
    w1 = (torch.randn(256, 64, device=dev) / 8).requires_grad_(True)
    w2 = (torch.randn(64, 256, device=dev) / 16).requires_grad_(True)
    tokens = torch.randint(64, (4, 60), device=dev)
    leaves = (x, nw, nb, w1, w2)

    def fn(x, nw, nb, w1, w2):
        y = x + act8.norm_mlp(x, nw, nb, w1, w2)
        return logprobs.cross_entropy(layer_norm.layer_norm(y, nw, nb, checkpoint="int8"), tokens)

    eager = fn(*leaves)
    want = torch.autograd.grad(eager, leaves)
    torch._dynamo.reset()
    loss = torch.compile(fn, backend="aot_eager", fullgraph=True)(*leaves)
    got = torch.autograd.grad(loss, leaves)
    assert torch.allclose(loss, eager, rtol=1e-6)
    for a, b in zip(got, want):
        assert _moved(a, b) < 1e-5
