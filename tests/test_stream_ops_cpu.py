"""CPU checks of the operators along the residual stream (token embedding,
residual with its norms, log probabilities from hidden states): argument checks
of the C ABI before any launch, shapes of the fake implementations, one graph
under torch.compile, refusals of tangents, and the LM's options."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from gmdn_amd import _native, embedding, logprobs, residual
from gmdn_amd import ops  # noqa: F401
from gmdn_amd.mixer import LM, Block, Branch

P = 0x1000
BF16, F32 = _native.DTYPE_BF16, _native.DTYPE_F32


def test_embedding_argument_checks():
    lib = _native.load()

    def fwd_(w=P, t=P, y=P, rows=4, V=10, d=8, ws=8, dtype=BF16):
        return lib.gmdn_embed_fwd(w, t, y, rows, V, d, ws, 1.0, dtype, None)

    assert fwd_(rows=-1) == 1 and fwd_(V=0) == 1 and fwd_(d=0) == 1 and fwd_(ws=-1) == 1 and fwd_(rows=1 << 31) == 1
    assert fwd_(dtype=5) == 2 and fwd_(V=(1 << 27) + 1) == 2 and fwd_(d=(1 << 20) + 1) == 2
    assert fwd_(rows=(1 << 31) - 1, d=1 << 10) == 2  # more pieces than a launch takes
    assert fwd_(w=None) == 1 and fwd_(t=None) == 1 and fwd_(y=None) == 1
    assert fwd_(w=None, t=None, y=None, rows=0) == 0

    need = lib.gmdn_embed_bwd_workspace_bytes(1000, 50, 64)
    assert need % 256 == 0 and need > 4 * 4 * 1000
    assert lib.gmdn_embed_bwd_workspace_bytes(0, 50, 64) == 0 and lib.gmdn_embed_bwd_workspace_bytes(10, 0, 64) == 0

    def bwd(dy=P, t=P, dw=P, ws=P, n=need, rows=1000, V=50, d=64, s=64, dtype=F32):
        return lib.gmdn_embed_bwd(dy, t, dw, ws, n, rows, V, d, s, 1.0, -1, dtype, None)

    assert bwd(n=need - 1) == 3 and bwd(ws=None) == 3
    assert bwd(dy=None) == 1 and bwd(t=None) == 1 and bwd(dw=None) == 1 and bwd(s=-1) == 1 and bwd(dtype=9) == 2
    assert bwd(rows=0, dw=None) == 1


def test_residual_argument_checks():
    lib = _native.load()

    def fwd_(x=P, y=P, w=P, p=None, g=None, s=None, r=P, z=P, rs=P, ps=None, rows=4, d=64, xs=64, eps=1e-6, xt=BF16,
             yt=BF16, wt=F32):
        return lib.gmdn_residual_norm_fwd(x, y, w, p, g, s, r, z, rs, ps, rows, d, xs, 64, 64, eps, xt, yt, wt, None)

    assert fwd_(d=0) == 1 and fwd_(rows=-1) == 1 and fwd_(xs=-1) == 1 and fwd_(eps=-1.0) == 1
    assert fwd_(eps=float("nan")) == 1
    assert fwd_(d=8193) == 2 and fwd_(xt=BF16, yt=F32) == 2 and fwd_(wt=7) == 2
    assert fwd_(x=None) == 1 and fwd_(y=None) == 1 and fwd_(r=None) == 1 and fwd_(z=None) == 1 and fwd_(rs=None) == 1
    assert fwd_(p=P) == 1  # a post norm keeps its statistic
    assert fwd_(x=None, rows=0) == 0
    need = lib.gmdn_residual_norm_bwd_workspace_floats(1000, 1024)
    assert need >= 3 * 1024 and lib.gmdn_residual_norm_bwd_workspace_floats(0, 64) == 0

    def bwd(r=P, y=P, w=P, p=None, g=None, s=None, rs=P, ps=None, dx=P, dy=P, dg=None, dw=P, dp=None, ds=None, ws=P,
            n=need, rows=1000, d=1024, xt=BF16, yt=BF16):
        return lib.gmdn_residual_norm_bwd(P, P, r, y, w, p, g, s, rs, ps, dx, dy, dg, dw, dp, ds, ws, n, rows, d, d, d, d, d, d,
                                          xt, yt, F32, None)

    assert bwd(ws=None) == 3 and bwd(n=1023) == 3
    assert bwd(r=None) == 1 and bwd(rs=None) == 1 and bwd(dx=None) == 1
    assert bwd(dy=None, xt=F32) == 1          # another type than dx's
    assert bwd(y=None) == 1                   # a bfloat16 r is formed again
    assert bwd(s=P, dy=None) == 1 and bwd(s=P, y=None) == 1
    assert bwd(g=P) == 1                      # the gate's gradient
    assert bwd(p=P) == 1                      # the post norm's statistic
    assert bwd(ds=P) == 1 and bwd(dp=P) == 1 and bwd(w=None) == 1  # a gradient of what is not there
    assert bwd(d=8193) == 2
    assert lib.gmdn_residual_norm_bwd(*[None] * 17, 0, 0, 64, 64, 64, 64, 64, 64, BF16, BF16, F32, None) == 0


def test_linear_logprobs_argument_checks():
    lib = _native.load()
    sizes = (100, 300, 64, 64, 64)

    def need(which, rows=100, V=300, d=64, xs=64, ws=64, dtype=BF16, x=P, w=P):
        return getattr(lib, f"gmdn_linear_logprobs_{which}_workspace_bytes")(x, w, rows, V, d, xs, ws, dtype)

    # operands that the products do not read where they are get a copy in the workspace
    for kw in (dict(d=65, xs=72, ws=72), dict(dtype=F32), dict(x=P + 2), dict(xs=65), dict(w=P + 8), dict(ws=1 << 23)):
        assert need("fwd", **kw) > need("fwd") and need("bwd", **kw) > need("bwd"), kw
    assert need("fwd", rows=0) == 0 and need("bwd", V=0) == 0
    # the logits' gradient comes in pieces: far less than all of it
    assert need("bwd", rows=1 << 17, V=1 << 17, d=64) < (3 << 30)

    def fwd_(x=P, w=P, t=P, lp=P, h=P, s=P, ws=P, n=need("fwd"), dims=sizes, dtype=BF16):
        return lib.gmdn_linear_logprobs_fwd(x, w, t, lp, h, s, ws, n, *dims, -100, dtype, None)

    assert fwd_(n=need("fwd") - 1) == 3 and fwd_(ws=None) == 3 and fwd_(ws=P + 8) == 1
    for name in ("x", "w", "t", "lp", "h", "s"):
        assert fwd_(**{name: None}) == 1, name
    assert fwd_(dims=(-1, 300, 64, 64, 64)) == 1 and fwd_(dims=(100, 0, 64, 64, 64)) == 1
    assert fwd_(dims=(100, 300, 0, 64, 64)) == 1 and fwd_(dims=(100, 300, 64, -1, 64)) == 1
    assert fwd_(dims=(100, (1 << 27) + 1, 64, 64, 64)) == 2 and fwd_(dims=(100, 300, (1 << 17) + 1, 64, 64)) == 2
    assert fwd_(dims=((1 << 27) + 1, 1, 64, 64, 64)) == 2 and fwd_(dims=(1 << 24, 1 << 27, 64, 64, 64)) == 2
    assert fwd_(dims=(1 << 28, 300, 1024, 1024, 1024)) == 2
    assert fwd_(dtype=4) == 2
    assert fwd_(x=None, dims=(0, 300, 64, 64, 64)) == 0

    def bwd(x=P, w=P, t=P, s=P, h=P, dx=P, dw=P, ws=P, n=need("bwd")):
        return lib.gmdn_linear_logprobs_bwd(x, w, t, s, h, None, None, dx, dw, ws, n, *sizes, -100, BF16, None)

    assert bwd(n=need("bwd") - 1) == 3 and bwd(ws=None) == 3 and bwd(ws=P + 8) == 1 and bwd(dx=None, dw=None) == 1
    for name in ("x", "w", "t", "s", "h"):
        assert bwd(**{name: None}) == 1, name


def test_fake_shapes():
    op = torch.ops.gmdn
    with FakeTensorMode():
        w = torch.empty(50, 24, device="cuda", dtype=torch.bfloat16)
        t = torch.empty(2, 5, device="cuda", dtype=torch.int64)
        y = op.embed_fwd(w, t)
        assert y.shape == (2, 5, 24) and y.dtype == w.dtype
        assert op.embed_bwd(y, t, 50, 1.0, -1).shape == (50, 24)
        x, v = torch.empty(2, 5, 24, device="cuda"), torch.empty(24, device="cuda")
        r, z, rstd, post = op.residual_norm_fwd(x, y, v, v, y, v, 1e-6)
        assert r.dtype == x.dtype and z.dtype == y.dtype and rstd.shape == post.shape == (2, 5)
        dx, dy, dw, dp, dg, ds = op.residual_norm_bwd(r, z, r, y, v, v, y, v, rstd, post)
        assert dx.dtype == x.dtype and dy.dtype == dg.dtype == y.dtype and dw.shape == dp.shape == ds.shape == (24,)
        r, z, rstd, post = op.residual_norm_fwd(x, x, None, None, None, None, 1e-6)
        assert post.numel() == 0
        grads = op.residual_norm_bwd(r, z, r, x, None, None, None, None, rstd, post)
        assert [g.numel() for g in grads] == [x.numel(), 0, 0, 0, 0, 0]
        lp, h, stats = op.linear_logprobs_fwd(y, w, t, -100)
        assert lp.shape == h.shape == (2, 5) and stats.shape == (2, 5, 2) and lp.dtype == torch.float32
        dx, dw = op.linear_logprobs_bwd(y, w, t, stats, h, lp, None, -100, True, False)
        assert dx.shape == y.shape and dw.numel() == 0


def _calls(device):
    def t(*shape):
        return torch.empty(*shape, device=device)

    x, w = t(4, 64), t(64)
    full = dict(post_weight=2, gate=3, scale=4)
    return {
        "embedding": (lambda k, a: embedding.embedding(k, a, 2.0), (t(9, 64),), ["embed_fwd", "embed_bwd"]),
        "add": (lambda k, *a: sum(v.sum() for v in residual.residual_norm(*a)), (x, x, w),
                ["residual_norm_fwd", "residual_norm_bwd"]),
        "residual": (lambda k, *a: sum(v.sum() for v in residual.residual_norm(
            *a[:2], a[5], **{n: a[i] for n, i in full.items()})), (x, x, w, x, w, w),
                     ["residual_norm_fwd", "residual_norm_bwd"]),
        "linear_logprobs": (lambda k, *a: sum(v.sum() for v in logprobs.linear_logprobs(*a, k)), (x, t(9, 64)),
                            ["linear_logprobs_fwd", "linear_logprobs_bwd"]),
        "linear_cross_entropy": (lambda k, *a: logprobs.linear_cross_entropy(*a, k), (x, t(9, 64)),
                                 ["linear_logprobs_fwd", "linear_logprobs_bwd"]),
    }


NAMES = ["embedding", "add", "residual", "linear_logprobs", "linear_cross_entropy"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_and_backward_trace_to_one_graph(name):
    call, inputs, wanted = _calls("meta")[name]

    def step(tokens, *xs):
        xs = [x.detach().requires_grad_() for x in xs]
        out = call(tokens, *xs)
        return torch.autograd.grad(out, xs, torch.empty_like(out))

    gm = make_fx(step, tracing_mode="symbolic")(torch.empty(4, dtype=torch.int64, device="meta"), *inputs)
    seen = [str(n.target).split(".")[1] for n in gm.graph.nodes if "gmdn" in str(n.target)]
    assert sorted(seen) == sorted(wanted)
    grads = next(n for n in gm.graph.nodes if n.op == "output").args[0]
    assert [g.meta["val"].shape for g in grads] == [x.shape for x in inputs]


@pytest.mark.parametrize("name", NAMES)
def test_compiles_to_one_graph(name):
    torch._dynamo.reset()
    with FakeTensorMode():
        call, inputs, _ = _calls("cuda")[name]
        tokens = torch.empty(4, dtype=torch.int64, device="cuda")
        out = torch.compile(call, backend="eager", fullgraph=True)(tokens, *(x.clone().requires_grad_() for x in inputs))
        assert out.requires_grad


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    with FakeTensorMode():
        call, inputs, _ = _calls("cuda")[name]
        tokens = torch.empty(4, dtype=torch.int64, device="cuda")
        for i in range(len(inputs)):
            with fwd.dual_level():
                given = [fwd.make_dual(x, x.clone()) if j == i else x for j, x in enumerate(inputs)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(tokens, *given)


@pytest.mark.parametrize("name", ["embed_bwd", "residual_norm_bwd", "linear_logprobs_bwd"])
def test_second_derivatives_raise(name):
    """Differentiating a backward operator's result raises rather than being zero."""
    kind = {"embed_bwd": "embedding", "residual_norm_bwd": "residual", "linear_logprobs_bwd": "linear_logprobs"}[name]
    call, inputs, _ = _calls("meta")[kind]
    xs = [x.clone().requires_grad_() for x in inputs]
    out = call(torch.empty(4, dtype=torch.int64, device="meta"), *xs)
    cot = torch.empty_like(out).requires_grad_()
    grads = torch.autograd.grad(out, xs, cot, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grads[0].sum(), cot)


def test_cpu_tensors_are_refused():
    x, t = torch.randn(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: embedding.embedding(t, x), lambda: residual.residual_norm(x, x),
                 lambda: logprobs.linear_logprobs(x, x, t)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_lm_options_and_parameters():
    """Operators in place of torch's change no parameter; a post norm, gates and
    scales add theirs.  What does not go together is refused."""
    def names(**kw):
        return {n: tuple(p.shape) for n, p in LM(50, 64, 1, 2, "delta", **kw).named_parameters()}

    plain = names()
    assert names(residual="fused", loss="linear", embedding="sorted", emb_scale=8.0) == plain
    more = names(residual="fused", post_norm=True, gated=True, layer_scale=0.1)
    assert set(more) - set(plain) == {f"blocks.0.join{i}.{n}" for i in (1, 2)
                                      for n in ("post.weight", "gate.weight", "gate.bias", "scale")}
    assert all(more[n] == plain[n] for n in plain)
    for bad in (dict(residual="sum"), dict(residual="fused", norm="layer"), dict(post_norm=True), dict(gated=True),
                dict(layer_scale=1.0), dict(embedding="hash"), dict(emb_scale=2.0), dict(loss="none")):
        with pytest.raises(ValueError):
            LM(50, 64, 1, 2, "delta", **bad)
    with pytest.raises(ValueError):
        embedding.embedding(torch.zeros(1, dtype=torch.int64), torch.zeros(5, 4), 1.0, 5)


def _fake_block(**kw):
    block = Block(64, 2, "delta", 64, residual="fused", **kw)
    block.mixer = nn.Linear(64, 64)  # a branch that is cheap to trace
    return block


def _ops_of(call):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    with Seen() as seen:
        call()
    return [n.split(".")[1] for n in seen.names if n.startswith("gmdn")]


def test_replaced_and_hooked_norms_are_called():
    """A norm that is not the plain module is called as it is, beside the
    operator without it."""
    with FakeTensorMode(), torch.device("cuda"):
        x = torch.empty(2, 64, 64)
        block = _fake_block()
        assert _ops_of(lambda: block(x)) == ["residual_norm_fwd"]
        called = []
        block.n2.register_forward_hook(lambda *a: called.append("n2"))
        assert _ops_of(lambda: block(x)) == ["residual_norm_fwd"] and called == ["n2"]
        block.n2 = nn.LayerNorm(64)
        assert _ops_of(lambda: block(x)) == ["residual_norm_fwd"]
        assert _ops_of(lambda: _fake_block(checkpoint="int8")(x)) == ["residual_norm_fwd", "gelu8_fwd", "act8_pack"]
        block = _fake_block(post_norm=True)
        assert _ops_of(lambda: block(x)) == ["residual_norm_fwd"] * 2
        block.join1.post.register_forward_hook(lambda *a: called.append("post"))
        assert _ops_of(lambda: block(x)) == ["residual_norm_fwd"] * 2 and called[-1] == "post"
        block.join1.post = nn.RMSNorm(64, eps=1e-3)  # another epsilon than the norm's
        assert _ops_of(lambda: block(x)) == ["residual_norm_fwd"] * 2


def test_lm_fuses_across_blocks_and_calls_hooked_ones():
    with FakeTensorMode(), torch.device("cuda"):
        idx = torch.empty(2, 64, dtype=torch.int64)
        lm = LM(50, 64, 3, 2, "delta", residual="fused", loss="linear", embedding="sorted")
        for blk in lm.blocks:
            blk.mixer = nn.Linear(64, 64)
        want = ["embed_fwd"] + ["residual_norm_fwd"] * 6
        assert _ops_of(lambda: lm(idx)) == want
        assert _ops_of(lambda: lm(idx, idx)) == want + ["linear_logprobs_fwd"]
        assert lm(idx, idx)[0] is None and lm(idx)[0].shape == (2, 64, 50)
        assert _ops_of(lambda: lm.score(idx)) == want + ["linear_logprobs_fwd"]
        assert _ops_of(lambda: lm.score(idx, top=3)) == want + ["logprobs_fwd"]
        called = []
        lm.blocks[1].register_forward_hook(lambda *a: called.append(1))
        assert _ops_of(lambda: lm(idx)) == ["embed_fwd"] + ["residual_norm_fwd"] * 3 and called == [1]
        lm.lm_head.register_forward_hook(lambda *a: called.append(2))
        assert "logprobs_fwd" in _ops_of(lambda: lm(idx, idx)) and called[-1] == 2


def test_branch_without_parts_adds():
    branch = Branch(8, False, False, None)
    x, y = torch.randn(3, 8), torch.randn(3, 8)
    r, z = branch(x, y, y, None)
    assert torch.equal(r, x + y) and z is None
