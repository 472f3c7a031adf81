"""CPU checks of the LM's operators (layer norm, 8-bit checkpoints, token log
probabilities): argument checks of the C ABI before any launch, shapes of the
fake implementations, and the LM stack's options."""
import os
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "gmdn-gated-muon-deltanet_amd"))

from gmdn_amd import _native, act8, layer_norm, logprobs  # noqa: E402
from gmdn_amd import ops  # noqa: E402,F401
from gmdn_amd.mixer import LM, Block  # noqa: E402

P = 0x1000
BF16, F32 = _native.DTYPE_BF16, _native.DTYPE_F32


def _ln(lib, rows=4, d=64, xs=64, eps=1e-5, xt=BF16, yt=BF16, wt=F32, x=P, w=P, b=P, y=P, mean=P, q=None, s=None):
    return lib.gmdn_layer_norm_fwd(x, w, b, y, mean, P, q, s, rows, d, xs, eps, xt, yt, wt, None)


def test_layer_norm_argument_checks():
    lib = _native.load()
    assert _ln(lib, d=0) == 1 and _ln(lib, rows=-1) == 1
    assert _ln(lib, d=16385) == 2
    assert _ln(lib, xt=BF16, yt=F32) == 2 and _ln(lib, xt=7) == 2 and _ln(lib, wt=5) == 2
    assert _ln(lib, eps=-1.0) == 1 and _ln(lib, eps=float("nan")) == 1
    assert _ln(lib, x=None) == 1 and _ln(lib, y=None) == 1 and _ln(lib, mean=None) == 1
    assert _ln(lib, w=None) == 1            # a bias needs a weight
    assert _ln(lib, q=P) == 1               # a checkpoint needs both tensors
    assert _ln(lib, xs=-1) == 1
    assert _ln(lib, rows=0, x=None) == 0    # nothing to do
    ws = lib.gmdn_layer_norm_bwd_workspace_floats(1000, 1024)
    assert ws > 0 and ws % (2 * 1024) == 0 and lib.gmdn_layer_norm_bwd_workspace_floats(0, 64) == 0

    def bwd(x=P, q=None, s=None, w=P, dw=P, ws_ptr=P, n=ws, rows=1000, d=1024):
        return lib.gmdn_layer_norm_bwd(P, x, q, s, w, P, P, P, dw, dw, ws_ptr, n, rows, d, d, d, BF16, BF16, F32, None)

    assert bwd(n=ws - 1) == 3 and bwd(ws_ptr=None) == 3
    assert bwd(x=None) == 1 and bwd(q=P, s=P) == 1 and bwd(dw=None) == 1 and bwd(x=None, q=P) == 1
    assert bwd(d=20000) == 2
    assert bwd(w=None, dw=None, ws_ptr=None, n=0, rows=0) == 0
    assert lib.gmdn_layer_norm8_rebuild(P, P, None, P, P, P, P, 4, 64, BF16, F32, None) == 1
    assert lib.gmdn_layer_norm8_rebuild(P, None, P, P, P, P, P, 4, 64, BF16, F32, None) == 1
    assert lib.gmdn_layer_norm8_rebuild(None, None, P, P, P, P, P, 0, 64, BF16, F32, None) == 0


def test_act8_argument_checks():
    lib = _native.load()
    assert [lib.gmdn_act8_groups(d) for d in (0, 1, 128, 129, 4096)] == [0, 1, 1, 2, 32]
    assert lib.gmdn_act8_pack(P, P, P, 4, 0, 64, BF16, None) == 1
    assert lib.gmdn_act8_pack(P, P, P, 4, 1 << 31, 64, BF16, None) == 1
    assert lib.gmdn_act8_pack(P, P, P, 4, 64, -1, BF16, None) == 1
    assert lib.gmdn_act8_pack(P, P, P, 4, 64, 64, 3, None) == 2
    assert lib.gmdn_act8_pack(P, None, P, 4, 64, 64, BF16, None) == 1
    assert lib.gmdn_act8_pack(None, None, None, 0, 64, 64, BF16, None) == 0
    assert lib.gmdn_act8_unpack(P, P, None, 4, 64, BF16, None) == 1
    assert lib.gmdn_gelu8_fwd(P, None, P, P, 4, 64, 64, BF16, None) == 1
    assert lib.gmdn_gelu8_fwd(P, P, P, None, 4, 64, 64, BF16, None) == 1
    assert lib.gmdn_gelu8_bwd(None, P, P, P, None, 4, 64, 64, BF16, None) == 1
    assert lib.gmdn_gelu8_bwd(None, None, None, None, None, 0, 64, 64, F32, None) == 0


def test_logprobs_argument_checks():
    lib = _native.load()

    def fwd(rows=4, V=100, stride=100, top=0, dtype=BF16, logits=P, topp=P, stats=P, ws=None, n=0):
        return lib.gmdn_logprobs_fwd(logits, P, P, P, topp, topp, stats, ws, n, rows, V, stride, top, -100, dtype, None)

    need = lib.gmdn_logprobs_fwd_workspace_bytes(1, 1 << 17, 20)
    assert need > 0 and lib.gmdn_logprobs_fwd_workspace_bytes(4096, 1 << 17, 20) == 0
    assert fwd(rows=1, V=1 << 17, top=20) == 3 and fwd(rows=1, V=1 << 17, top=20, ws=P, n=need - 1) == 3

    assert fwd(V=0) == 1 and fwd(rows=-1) == 1 and fwd(stride=-1) == 1 and fwd(rows=1 << 31) == 1
    assert fwd(top=-1) == 1 and fwd(V=8, top=9) == 1 and fwd(top=33) == 2
    assert fwd(dtype=9) == 2 and fwd(V=(1 << 30) + 1) == 2
    assert fwd(logits=None) == 1 and fwd(stats=None) == 1 and fwd(top=2, topp=None) == 1
    assert fwd(rows=0, logits=None) == 0

    def bwd(dlogits=P, topp=None, dtop=None, top=0):
        return lib.gmdn_logprobs_bwd(P, P, P, P, topp, None, None, dtop, dlogits, 4, 100, 100, top, -100, BF16, None)

    assert bwd(dlogits=None) == 1 and bwd(dtop=P, top=3) == 1


def test_fake_shapes():
    with FakeTensorMode():
        x = torch.empty(2, 5, 300, device="cuda")
        w = torch.empty(300, device="cuda")
        y, mean, rstd, q, scale = torch.ops.gmdn.layer_norm_fwd(x, w, w, 1e-5, torch.bfloat16, True)
        assert y.shape == x.shape and y.dtype == torch.bfloat16 and mean.shape == rstd.shape == (2, 5)
        assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == (2, 5, 3)
        assert torch.ops.gmdn.layer_norm_fwd(x, None, None, 1e-5, x.dtype, False)[3].numel() == 0
        dx, dw, db = torch.ops.gmdn.layer_norm_bwd(y, x, w, mean, rstd)
        assert dx.dtype == x.dtype and dw.shape == db.shape == (300,)
        dx, dw, db = torch.ops.gmdn.layer_norm8_bwd(y, q, scale, None, mean, rstd, torch.float32)
        assert dx.dtype == torch.float32 and dw.numel() == db.numel() == 0
        assert torch.ops.gmdn.layer_norm8_rebuild(q, scale, w, w, mean, rstd, torch.float32).dtype == torch.float32
        assert torch.ops.gmdn.act8_unpack(*torch.ops.gmdn.act8_pack(x), torch.bfloat16).dtype == torch.bfloat16
        a, q, scale = torch.ops.gmdn.gelu8_fwd(x)
        dh, again = torch.ops.gmdn.gelu8_bwd(a, q, scale, False)
        assert dh.shape == x.shape and again.numel() == 0
        tokens = torch.empty(2, 5, dtype=torch.int64, device="cuda")
        l, h, tl, tt, stats = torch.ops.gmdn.logprobs_fwd(x, tokens, 4, -100)
        assert l.shape == h.shape == (2, 5) and tl.shape == tt.shape == (2, 5, 4) and tt.dtype == torch.int64
        assert torch.ops.gmdn.logprobs_bwd(x, tokens, stats, h, tt, l, None, None, -100).shape == x.shape


@pytest.mark.parametrize("which", ["norm", "gelu", "lp"])
def test_compiles_to_one_graph(which):
    """torch.compile traces the operators, forward and backward, in one graph."""
    seen = []

    def backend(gm, inputs):
        seen.append([str(n.target) for n in gm.graph.nodes if n.op == "call_function"])
        return gm.forward

    def fn(x, t):
        if which == "norm":
            return layer_norm.layer_norm(x, checkpoint="int8")
        if which == "gelu":
            return act8.gelu(x)
        return logprobs.token_logprobs(x, t, 3).logprob

    torch._dynamo.reset()
    with FakeTensorMode():
        x = torch.empty(4, 64, device="cuda", requires_grad=True)
        t = torch.empty(4, dtype=torch.int64, device="cuda")
        out = torch.compile(fn, backend=backend, fullgraph=True)(x, t)
        assert out.requires_grad
    assert len(seen) == 1
    name = {"norm": "layer_norm_fwd", "gelu": "gelu8_fwd", "lp": "logprobs_fwd"}[which]
    assert any(name in s for s in seen[0])


def test_lm_options_keep_the_parameters():
    """norm="rms" with any checkpoint has the reference's parameters; layer norm
    adds a bias to each norm.  Unknown names are refused."""
    plain = {n: p.shape for n, p in LM(50, 64, 1, 2, "muon").named_parameters()}
    kept = {n: p.shape for n, p in LM(50, 64, 1, 2, "muon", checkpoint="int8", loss="logprobs").named_parameters()}
    assert plain == kept
    layer = {n: p.shape for n, p in LM(50, 64, 1, 2, "muon", norm="layer").named_parameters()}
    assert set(layer) - set(plain) == {"blocks.0.n1.bias", "blocks.0.n2.bias", "norm_f.bias"}
    for bad in (dict(norm="batch"), dict(checkpoint="int4"), dict(loss="mean")):
        with pytest.raises(ValueError):
            LM(50, 64, 1, 2, "muon", **bad)
    with pytest.raises(ValueError):
        Block(64, 2, "muon", 64, checkpoint="fp8")


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 8)
    for call in (lambda: layer_norm.layer_norm(x), lambda: act8.pack(x), lambda: act8.gelu(x),
                 lambda: logprobs.token_logprobs(x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
