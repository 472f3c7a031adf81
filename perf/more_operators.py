"""The operators along an LM's residual stream beside its blocks: the token
embedding with its gradient, a branch's way back into the stream with the norm
that follows it, and the tied head's log probabilities without the logits.

A case is a dict of plain values; ``kind`` selects the operator and ``mode``
how it is used ("forward" or "score" without, "train" with the backward):

* ``embed``    -- rows of the table at given tokens, times ``scale``.  "train":
  the table's gradient too, zeros where no token asked for a row.
* ``residual`` -- r = x + s * sigmoid(gate) * post(y) and z = norm(r): ``x`` the
  stream, ``y`` a branch's output, ``post`` and ``norm`` RMS norms with weights;
  ``full`` has the post norm, the gate (logits, (rows, D)) and the scale s (D),
  "post" the post norm and the scale, "add" none of them.  "train": the
  gradients of all of them.
* ``head``     -- log probability of given tokens and entropy of
  softmax(x W^T) for each row of x.  "train": the gradients of x and W.

``dtype`` is the type of the table, the stream or the head's operands;
``branch`` that of a branch's output, its gate and the norm's result.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.abspath("gmdn-gated-muon-deltanet_amd")
EPS = 1e-6
IGNORE = -100
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decoding step's lookup for eight sequences: latency
        dict(name="embed_token", kind="embed", mode="forward", rows=8, V=32000, D=1024, dtype="bf16", scaled=False, pad=0.0),
        # the 12-layer LM's step: B = 8, T = 2048 tokens of a vocabulary of 32000
        dict(name="embed_lm_train", kind="embed", mode="train", rows=16384, V=32000, D=1024, dtype="bf16", scaled=False, pad=0.0),
        # a padded batch in float32 at an odd width, scaled by sqrt(D): half of its tokens are one padding token
        dict(name="embed_padded_train", kind="embed", mode="train", rows=4099, V=32003, D=1001, dtype="f32", scaled=True, pad=0.5),
        # a large table
        dict(name="embed_wide_train", kind="embed", mode="train", rows=16384, V=131072, D=4096, dtype="bf16", scaled=True, pad=0.0),
        # one decoding step's residual and norm for eight sequences: latency
        dict(name="residual_token", kind="residual", mode="forward", rows=8, D=1024, dtype="bf16", branch="bf16", parts="add"),
        # a block of the 12-layer LM: float32 stream, bfloat16 branches
        dict(name="residual_lm_train", kind="residual", mode="train", rows=16384, D=1024, dtype="f32", branch="bf16", parts="add"),
        # a wide model's with everything on it
        dict(name="residual_full_train", kind="residual", mode="train", rows=8192, D=8192, dtype="bf16", branch="bf16", parts="full"),
        # an odd width in float32
        dict(name="residual_odd_train", kind="residual", mode="train", rows=4099, D=1001, dtype="f32", branch="f32", parts="post"),
        # a decoding step's chosen tokens, eight sequences
        dict(name="head_decode", kind="head", mode="score", rows=8, V=32000, D=1024, dtype="bf16"),
        # a small model's loss
        dict(name="head_small_train", kind="head", mode="train", rows=512, V=257, D=256, dtype="f32"),
        # odd everything in float32
        dict(name="head_odd_train", kind="head", mode="train", rows=1021, V=32003, D=1001, dtype="f32"),
        # the 12-layer LM's loss: every token of a step over its whole vocabulary
        dict(name="head_lm_train", kind="head", mode="train", rows=16384, V=32000, D=1024, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _size(rng, lo, hi, unit):
    """Over the whole range; half of the time a multiple of ``unit``."""
    return rng.choice([_log_int(rng, lo, hi), unit * _log_int(rng, -(-lo // unit), hi // unit)])


def draw(rng):
    kind = rng.choice(["embed", "residual", "head"])
    if kind == "embed":
        V, D = _size(rng, 64, 131072, 64), _size(rng, 16, 8192, 64)
        V = min(V, (1 << 29) // D)
        return dict(kind=kind, mode=rng.choice(["forward", "train", "train"]), rows=_log_int(rng, 1, min(32768, (1 << 26) // D)),
                    V=V, D=D, dtype=rng.choice(["bf16", "f32"]) if V * D <= 1 << 28 else "bf16",
                    scaled=rng.random() < 0.5, pad=rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.9), 2)]))
    if kind == "residual":
        D = _size(rng, 16, 8192, 128)
        dtype, branch = rng.choice([("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
        most = (1 << 26) // D if dtype == "bf16" else (1 << 25) // D
        return dict(kind=kind, mode=rng.choice(["forward", "train", "train"]), rows=_log_int(rng, 1, min(32768, most)), D=D,
                    dtype=dtype, branch=branch, parts=rng.choice(["add", "post", "full"]))
    dtype, mode = rng.choice(["bf16", "f32"]), rng.choice(["score", "train"])
    V, D = _size(rng, 64, 131072, 64), _size(rng, 16, 4096, 64)
    # products of at most the 12-layer LM's work, a quarter of it in float32
    most = (1 << 39 if dtype == "bf16" else 1 << 37) // (V * D)
    return dict(kind=kind, mode=mode, rows=_log_int(rng, 1, max(1, min(16384, most, (1 << 29) // V))), V=V, D=D, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)
    return x.mul_(scale) if scale != 1.0 else x


def _tokens(g, rows, V):
    """As text has them: a token's frequency falls with its rank, 1 / (rank + 1)."""
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    return ((V + 1.0) ** u - 1).long().clamp_(0, V - 1)


def _embed_inputs(c, g):
    rows, V, D, dt = c["rows"], c["V"], c["D"], _TYPES[c["dtype"]]
    tokens = _tokens(g, rows, V)
    if c["pad"]:
        tokens[torch.rand(rows, generator=g, device="cuda") < c["pad"]] = V - 1
    s = {"weight": _randn(g, (V, D), dt, 0.02), "tokens": tokens, "scale": math.sqrt(D) if c["scaled"] else 1.0}
    if c["mode"] == "train":
        s["dy"] = _randn(g, (rows, D), dt, 1e-3)
    return s


def _residual_inputs(c, g):
    rows, D, dt, bt = c["rows"], c["D"], _TYPES[c["dtype"]], _TYPES[c["branch"]]
    channel = 1 + 9 * (torch.rand(D, generator=g, device="cuda") < 0.01)  # a few are larger in every row
    s = {"x": _randn(g, (rows, D), dt).mul_(channel.to(dt)), "y": _randn(g, (rows, D), bt, 0.5), "eps": EPS,
         "weight": 1 + 0.1 * _randn(g, (D,), torch.float32), "post": None, "gate": None, "scale": None}
    if c["parts"] != "add":
        s["post"] = 1 + 0.1 * _randn(g, (D,), torch.float32)
        s["scale"] = 0.5 + 0.1 * _randn(g, (D,), torch.float32)
    if c["parts"] == "full":
        s["gate"] = _randn(g, (rows, D), bt)
    if c["mode"] == "train":
        s["dr"], s["dz"] = _randn(g, (rows, D), dt, 1e-3), _randn(g, (rows, D), bt, 1e-3)
    return s


def _head_inputs(c, g):
    rows, V, D, dt = c["rows"], c["V"], c["D"], _TYPES[c["dtype"]]
    weight = _randn(g, (V, D), dt, 1.5 / math.sqrt(D))
    tokens = _tokens(g, rows, V)
    # what a trained model gives: a token's hidden state leans towards its row of the head
    lean = 3 * torch.rand(rows, 1, generator=g, device="cuda")
    x = (_randn(g, (rows, D), torch.float32) + lean * weight[tokens].float()).to(dt)
    tokens[torch.rand(rows, generator=g, device="cuda") < 0.05] = IGNORE  # padding
    s = {"x": x, "weight": weight, "tokens": tokens}
    if c["mode"] == "train":
        s["dlogprob"] = _randn(g, (rows,), torch.float32, 1.0 / rows)    # advantages
        s["dentropy"] = torch.full((rows,), 0.01 / rows, device="cuda")   # an entropy bonus
    return s


_INPUTS = {"embed": _embed_inputs, "residual": _residual_inputs, "head": _head_inputs}


def prepare(case, seed):
    return dict(_INPUTS[case["kind"]](case, _gen(seed)), kind=case["kind"], mode=case["mode"])


# ------------------------------------------------------------------ the framework's operators
_gmdn = None


def _ops():
    """torch.ops.gmdn, the framework's operators."""
    global _gmdn
    if _gmdn is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        from gmdn_amd import ops
        ops.ensure()
        _gmdn = torch.ops.gmdn
    return _gmdn


def _run_own(s):
    op, kind, train = _ops(), s["kind"], s["mode"] == "train"
    if kind == "embed":
        y = op.embed_fwd(s["weight"], s["tokens"], s["scale"])
        if not train:
            return {"y": y}
        return {"y": y, "dweight": op.embed_bwd(s["dy"], s["tokens"], s["weight"].shape[0], s["scale"], -1)}
    if kind == "residual":
        parts = s["weight"], s["post"], s["gate"], s["scale"]
        r, z, rstd, post_rstd = op.residual_norm_fwd(s["x"], s["y"], *parts, s["eps"])
        if not train:
            return {"r": r, "z": z}
        # the backward takes x, but of a float32 stream with nothing but the sum r
        plain = s["post"] is None and s["gate"] is None and s["scale"] is None
        stream = r if plain and r.dtype == torch.float32 else s["x"]
        dx, dy, dw, dpost, dgate, dscale = op.residual_norm_bwd(s["dr"], s["dz"], stream, s["y"], *parts, rstd, post_rstd)
        out = {"r": r, "z": z, "dx": dx, "dy": dy if dy.numel() else dx, "dweight": dw}
        if s["post"] is not None:
            out.update(dpost=dpost, dscale=dscale)
        return dict(out, dgate=dgate) if s["gate"] is not None else out
    lp, entropy, stats = op.linear_logprobs_fwd(s["x"], s["weight"], s["tokens"], IGNORE)
    if not train:
        return {"logprob": lp, "entropy": entropy}
    dx, dw = op.linear_logprobs_bwd(s["x"], s["weight"], s["tokens"], stats, entropy, s["dlogprob"], s["dentropy"], IGNORE,
                                    True, True)
    return {"logprob": lp, "entropy": entropy, "dx": dx, "dweight": dw}


# ------------------------------------------------------------------ the plain form
def _plain_embed(s):
    w, tokens = s["weight"], s["tokens"]
    out = {"y": (w[tokens].float() * s["scale"]).to(w.dtype)}
    if s["mode"] == "train":
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        dw.index_add_(0, tokens, s["dy"].float() * s["scale"])
        out["dweight"] = dw.to(w.dtype)
    return out


def _rms(x, eps):
    return torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)


def _plain_residual(s):
    x, y, w = s["x"].float(), s["y"].float(), s["weight"]
    post, gate, scale, eps = s["post"], s["gate"], s["scale"], s["eps"]
    ry = _rms(y, eps) if post is not None else None
    yh = y * ry if post is not None else y
    n = yh * post if post is not None else y
    sig = torch.sigmoid(gate.float()) if gate is not None else None
    mult = 1.0 if sig is None else sig
    mult = mult if scale is None else mult * scale
    r = x + mult * n
    rr = _rms(r, eps)
    rh = r * rr
    out = {"r": r.to(s["x"].dtype), "z": (rh * w).to(s["y"].dtype)}
    if s["mode"] != "train":
        return out
    dz = s["dz"].float()
    g = dz * w
    dx = s["dr"].float() + rr * (g - rh * (g * rh).mean(-1, keepdim=True))
    dn = dx * mult
    dy = dn
    if post is not None:
        g = dn * post
        dy = ry * (g - yh * (g * yh).mean(-1, keepdim=True))
    out.update(dx=dx.to(s["x"].dtype), dy=dy.to(s["y"].dtype), dweight=(dz * rh).sum(0))
    if post is not None:
        out.update(dpost=(dn * yh).sum(0), dscale=((dx * n) if sig is None else dx * sig * n).sum(0))
    if sig is not None:
        out["dgate"] = (dx * scale * n * sig * (1 - sig)).to(gate.dtype)
    return out


def _plain_head(s):
    x, w, tokens = s["x"].float(), s["weight"].float(), s["tokens"]
    logits = x @ w.t()
    peak = logits.amax(-1, keepdim=True)
    logp = logits - peak
    del logits
    logp -= torch.log(torch.exp(logp).sum(-1, keepdim=True))
    p = torch.exp(logp)
    entropy = -(p * logp).sum(-1)
    kept = tokens != IGNORE
    at = torch.where(kept, tokens, torch.zeros_like(tokens))[:, None]
    lp = torch.where(kept, logp.gather(1, at)[:, 0], torch.zeros_like(entropy))
    out = {"logprob": lp, "entropy": entropy}
    if s["mode"] == "train":
        gl, gh = (s["dlogprob"] * kept)[:, None], s["dentropy"][:, None]
        d = logp.add_(entropy[:, None]).mul_(-gh).sub_(gl).mul_(p)  # -p (gl + gh (log p + entropy))
        d.scatter_add_(1, at, gl)
        out.update(dx=(d @ w).to(s["x"].dtype), dweight=(d.t() @ x).to(s["weight"].dtype))
    return out


_PLAIN = {"embed": _plain_embed, "residual": _plain_residual, "head": _plain_head}


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    size, train = _SIZE[c["dtype"]], c["mode"] == "train"
    n = c["rows"] * c["D"]
    if c["kind"] == "embed":
        # the tokens and their rows read, y written; dy read, the whole gradient written
        forward = 8 * c["rows"] + 2 * n * size
        if not train:
            return {"bytes": forward, "flops": n}
        return {"bytes": forward + 8 * c["rows"] + (n + c["V"] * c["D"]) * size, "flops": 3 * n}
    if c["kind"] == "residual":
        # x, y and a gate read, r and z written; dr, dz, r, y and a gate read, dx, dy and a gate's written
        branch, vectors = _SIZE[c["branch"]], 1 if c["parts"] == "add" else 3
        gate = n * branch if c["parts"] == "full" else 0
        forward = 2 * n * (size + branch) + gate + 4 * vectors * c["D"]
        if not train:
            return {"bytes": forward, "flops": 14 * n}
        return {"bytes": forward + 3 * n * (size + branch) + 2 * gate + 8 * vectors * c["D"], "flops": 48 * n}
    # x and W read, 8 bytes a row out; both again and their gradients; three products
    table = (n + c["V"] * c["D"]) * size
    product = 2 * n * c["V"]
    if not train:
        return {"bytes": table + 16 * c["rows"], "flops": product}
    return {"bytes": 3 * table + 40 * c["rows"], "flops": 3 * product}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_embed(s):
    y = s["weight"].index_select(0, s["tokens"]).double() * s["scale"]
    if s["mode"] != "train":
        return {"y": y}
    # sums over the tokens in their sorted order, by differences at the ends of equal runs
    V, D = s["weight"].shape
    order = torch.argsort(s["tokens"], stable=True)
    run_of, counts = torch.unique_consecutive(s["tokens"][order], return_counts=True)
    dw = torch.zeros(V, D, dtype=torch.float64, device=y.device)
    dw[run_of] = torch.segment_reduce(s["dy"][order].double(), "sum", lengths=counts, axis=0) * s["scale"]
    return {"y": y, "dweight": dw}


def _exact_residual(s):
    names = [n for n in ("x", "y", "weight", "post", "gate", "scale") if s[n] is not None]
    train = s["mode"] == "train"
    leaf = {n: s[n].double().requires_grad_(train) for n in names}
    branch = leaf["y"]
    if "post" in leaf:
        branch = branch / (branch.square().mean(1, keepdim=True) + s["eps"]).sqrt() * leaf["post"]
    if "gate" in leaf:
        branch = branch / (1 + torch.exp(-leaf["gate"]))
    if "scale" in leaf:
        branch = branch * leaf["scale"]
    r = leaf["x"] + branch
    z = r / (r.square().mean(1, keepdim=True) + s["eps"]).sqrt() * leaf["weight"]
    out = {"r": r.detach(), "z": z.detach()}
    if train:
        grads = torch.autograd.grad([r, z], [leaf[n] for n in names], [s["dr"].double(), s["dz"].double()])
        out.update(("d" + n, g) for n, g in zip(names, grads))
    return out


def _exact_head(s):
    rows, V = s["x"].shape[0], s["weight"].shape[0]
    x, w = s["x"].double(), s["weight"].double()
    lp, entropy, dx = [], [], []
    dw = torch.zeros_like(w) if s["mode"] == "train" else None
    step = max(1, (1 << 27) // V)
    for a in range(0, rows, step):  # a part of the rows at a time
        part = slice(a, a + step)
        logp = torch.log_softmax(x[part].mm(w.t()), 1)
        p = logp.exp()
        entropy.append(torch.special.entr(p).sum(1))
        tokens = s["tokens"][part]
        kept = tokens >= 0
        at = tokens.clamp_min(0)[:, None]
        lp.append(torch.where(kept, logp.gather(1, at)[:, 0], 0.0))
        if dw is None:
            continue
        gl = torch.where(kept, s["dlogprob"][part].double(), 0.0)[:, None]
        gh = s["dentropy"][part].double()[:, None]
        d = gh * (torch.special.entr(p) - p * entropy[-1][:, None]) - gl * p
        d = d + torch.zeros_like(p).scatter_(1, at, 1.0) * gl
        dx.append(d.mm(w))
        dw += d.t().mm(x[part])
    out = {"logprob": torch.cat(lp), "entropy": torch.cat(entropy)}
    return dict(out, dx=torch.cat(dx), dweight=dw) if dw is not None else out


_EXACT = {"embed": _exact_embed, "residual": _exact_residual, "head": _exact_head}


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))
