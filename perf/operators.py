"""The operators of an LM's training and scoring step around the mixer: layer
norm with its backward pass, activation checkpoints in 8 bits, and the log
probabilities of given tokens.

A case is a dict of plain values; ``kind`` selects the operator and ``mode``
how it is used:

* ``norm``  -- layer norm over (rows, D).  "forward": y.  "train": forward, and
  the backward from the saved mean and 1 / deviation: dx, dweight, dbias.
* ``act8``  -- activation checkpoints: int8 values with a float32 scale for
  each group of 128 consecutive values of a row.
  "pack": the checkpoint of a tensor and what it reads back as.
  "gelu": GELU that keeps its input in 8 bits: the output, and from the
  checkpoint the input's gradient and the output again (for the weight gradient
  of the product behind it).
  "norm": layer norm that keeps its input in 8 bits: y, and from the
  checkpoint y again, dx, dweight, dbias.
* ``lp``    -- log probabilities of given tokens.  "score": log probability,
  entropy, and the ``top`` likeliest tokens with theirs.  "train": log
  probability, entropy and the logits' gradient.

``dtype`` is the activations' or logits' type, ``out`` that of a norm's output.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.abspath("gmdn-gated-muon-deltanet_amd")
GROUP = 128                             # values of a checkpoint's group
STEP = float.fromhex("0x1.020406p-7")   # scale / amax: the float32 below 1 / 127
TINY = 2.0 ** -100                      # a group below it is kept as zeros
EPS = 1e-5
IGNORE = -100
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decoding step's norm for eight sequences: latency
        dict(name="norm_token", kind="norm", mode="forward", rows=8, D=1024, dtype="bf16", out="bf16"),
        # a block's pre-norm in the 12-layer LM's step: float32 residual stream, bfloat16 into the projection
        dict(name="norm_lm_train", kind="norm", mode="train", rows=16384, D=1024, dtype="f32", out="bf16"),
        # a wide model's training norm
        dict(name="norm_wide_train", kind="norm", mode="train", rows=8192, D=8192, dtype="bf16", out="bf16"),
        # an odd width in float32: rows at every alignment
        dict(name="norm_odd_train", kind="norm", mode="train", rows=4099, D=1001, dtype="f32", out="f32"),
        # the input of a projection kept in 8 bits between the passes
        dict(name="act8_lm_pack", kind="act8", mode="pack", rows=16384, D=1024, dtype="bf16"),
        # the smallest configuration's MLP
        dict(name="act8_small_gelu", kind="act8", mode="gelu", rows=256, D=512, dtype="f32"),
        # the 12-layer LM's MLP activation, 4 x 1024 wide
        dict(name="act8_lm_gelu", kind="act8", mode="gelu", rows=16384, D=4096, dtype="bf16"),
        # its pre-norm, keeping the residual stream in 8 bits
        dict(name="act8_lm_norm", kind="act8", mode="norm", rows=16384, D=1024, dtype="f32", out="bf16"),
        # a decoding step's chosen tokens with 20 alternatives
        dict(name="lp_decode", kind="lp", mode="score", rows=8, V=32000, pad=0, dtype="bf16", top=20, masked=False),
        # scoring under vocabulary masks, some of which leave a few tokens or none; padded rows
        dict(name="lp_masked_score", kind="lp", mode="score", rows=1021, V=32003, pad=61, dtype="f32", top=8, masked=True),
        # a small vocabulary's training loss
        dict(name="lp_small_train", kind="lp", mode="train", rows=512, V=257, pad=0, dtype="f32", top=0, masked=False),
        # the 12-layer LM's loss: every token of a step over its whole vocabulary
        dict(name="lp_lm_train", kind="lp", mode="train", rows=16384, V=32000, pad=0, dtype="bf16", top=0, masked=False),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def draw(rng):
    kind = rng.choice(["norm", "act8", "lp"])
    if kind == "lp":
        V = rng.choice([_log_int(rng, 64, 131072), 8 * _log_int(rng, 8, 16384)])
        mode = rng.choice(["score", "train"])
        most = (1 << 26 if mode == "score" else 1 << 28) // V
        return dict(kind=kind, mode=mode, rows=_log_int(rng, 1, min(16384, most)), V=V,
                    pad=rng.choice([0, 0, _log_int(rng, 1, 64)]), dtype=rng.choice(["bf16", "f32"]),
                    top=rng.choice([1, 5, 20, 32]) if mode == "score" else 0, masked=rng.random() < 0.4)
    D = rng.choice([_log_int(rng, 16, 8192), 128 * _log_int(rng, 1, 64)])
    rows = _log_int(rng, 1, min(32768, (1 << 26) // D))
    dtype, out = rng.choice([("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
    if kind == "norm":
        return dict(kind=kind, mode=rng.choice(["forward", "train"]), rows=rows, D=D, dtype=dtype, out=out)
    mode = rng.choice(["pack", "gelu", "norm"])
    case = dict(kind=kind, mode=mode, rows=rows, D=D, dtype=dtype)
    return dict(case, out=out) if mode == "norm" else case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)
    return x.mul_(scale) if scale != 1.0 else x


def _rows_data(c, g):
    """Residual-stream rows: unit noise beside a few channels that are larger in every row."""
    x = _randn(g, (c["rows"], c["D"]), _TYPES[c["dtype"]])
    channel = 1 + 9 * (torch.rand(c["D"], generator=g, device="cuda") < 0.01)
    return x.mul_(channel.to(x.dtype)).add_(0.1)


def _norm_inputs(c, g):
    s = {"x": _rows_data(c, g), "eps": EPS, "out": _TYPES[c["out"]],
         "weight": 1 + 0.1 * _randn(g, (c["D"],), torch.float32), "bias": 0.1 * _randn(g, (c["D"],), torch.float32)}
    if c["mode"] != "forward":
        s["dy"] = _randn(g, (c["rows"], c["D"]), _TYPES[c["out"]], 1e-3)
    return s


def _lp_inputs(c, g):
    rows, V, dt = c["rows"], c["V"], _TYPES[c["dtype"]]
    logits = _randn(g, (rows, V + c["pad"]), dt, 2.0)[:, :V]
    tokens = torch.randint(V, (rows,), generator=g, device="cuda")
    # what a trained model gives: the token that follows is often among the likeliest
    at = tokens[:, None]
    lift = 8 * torch.rand(rows, 1, generator=g, device="cuda")
    logits.scatter_(1, at, (logits.gather(1, at).float() + lift).to(dt))
    if c["masked"]:
        # each row its own share of allowed tokens; one row in eight a handful, one in sixty-four none
        keep = torch.rand(rows, 1, generator=g, device="cuda")
        kind = torch.randint(64, (rows, 1), generator=g, device="cuda")
        keep = torch.where(kind < 8, torch.full_like(keep, 5.0 / V), keep)
        keep = torch.where(kind == 8, torch.zeros_like(keep), keep)
        logits.masked_fill_(torch.rand(rows, V, generator=g, device="cuda") >= keep, -math.inf)
    tokens[torch.rand(rows, generator=g, device="cuda") < 0.05] = IGNORE  # padding
    s = {"logits": logits, "tokens": tokens, "top": c["top"]}
    if c["mode"] == "train":
        s["dlogprob"] = _randn(g, (rows,), torch.float32, 1.0 / rows)     # advantages
        s["dentropy"] = torch.full((rows,), 0.01 / rows, device="cuda")    # an entropy bonus
    return s


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "lp":
        s = _lp_inputs(c, g)
    elif c["kind"] == "norm" or c["mode"] == "norm":
        s = _norm_inputs(c, g)
    else:
        s = {"x": _rows_data(c, g)}
        if c["mode"] == "gelu":
            s["dy"] = _randn(g, (c["rows"], c["D"]), _TYPES[c["dtype"]], 1e-3)
    return dict(s, kind=c["kind"], mode=c["mode"])


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
    op, kind, mode = _ops(), s["kind"], s["mode"]
    if kind == "norm":
        y, mean, rstd, _, _ = op.layer_norm_fwd(s["x"], s["weight"], s["bias"], s["eps"], s["out"], False)
        if mode == "forward":
            return {"y": y}
        dx, dw, db = op.layer_norm_bwd(s["dy"], s["x"], s["weight"], mean, rstd)
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if kind == "act8":
        x = s["x"]
        if mode == "pack":
            q, scale = op.act8_pack(x)
            return {"x": op.act8_unpack(q, scale, x.dtype)}
        if mode == "gelu":
            y, q, scale = op.gelu8_fwd(x)
            dx, again = op.gelu8_bwd(s["dy"], q, scale, True)
            return {"y": y, "dx": dx, "again": again}
        y, mean, rstd, q, scale = op.layer_norm_fwd(x, s["weight"], s["bias"], s["eps"], s["out"], True)
        again = op.layer_norm8_rebuild(q, scale, s["weight"], s["bias"], mean, rstd, s["out"])
        dx, dw, db = op.layer_norm8_bwd(s["dy"], q, scale, s["weight"], mean, rstd, x.dtype)
        return {"y": y, "again": again, "dx": dx, "dweight": dw, "dbias": db}
    lp, entropy, top_lp, top, lse = op.logprobs_fwd(s["logits"], s["tokens"], s["top"], IGNORE)
    if mode == "score":
        return {"logprob": lp, "entropy": entropy, "top_logprobs": top_lp, "top_tokens": top}
    dlogits = op.logprobs_bwd(s["logits"], s["tokens"], lse, entropy, top, s["dlogprob"], s["dentropy"], None, IGNORE)
    return {"logprob": lp, "entropy": entropy, "dlogits": dlogits}


# ------------------------------------------------------------------ the plain form
def _norm_stats(x, eps):
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    return mean, torch.rsqrt((centred * centred).mean(-1, keepdim=True) + eps)


def _norm_grads(xhat, rstd, weight, dy):
    g = dy * weight
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0)


def _read_back(x):
    """What the 8-bit checkpoint of float32 rows reads back as, in float32."""
    rows, D = x.shape
    groups = -(-D // GROUP)
    v = torch.nn.functional.pad(x, (0, groups * GROUP - D)).view(rows, groups, GROUP)
    amax = v.abs().amax(-1, keepdim=True)
    zero, finite = amax < TINY, torch.isfinite(amax)
    inverse = torch.where(zero | ~finite, torch.zeros_like(amax), torch.div(torch.full_like(amax, 127.0), amax))
    scale = torch.where(zero, torch.zeros_like(amax), torch.where(finite, amax * STEP, torch.full_like(amax, math.nan)))
    q = torch.where(finite, torch.round(v * inverse), torch.zeros_like(v))
    return (q * scale).view(rows, groups * GROUP)[:, :D]


def _gelu(x):
    """GELU (with the normal distribution function) and its derivative."""
    cdf = 0.5 * torch.special.erfc(-x * math.sqrt(0.5))
    density = torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    return x * cdf, cdf + x * density


def _plain_lp(s):
    x = s["logits"].float()
    rows, V = x.shape
    peak = x.amax(-1, keepdim=True)
    empty = peak == -math.inf
    base = torch.where(empty, torch.zeros_like(peak), peak)
    total = torch.exp(x - base).sum(-1, keepdim=True)
    logp = x - base - torch.log(total)
    logp = torch.where(empty, torch.full_like(logp, -math.inf), logp)
    p = torch.exp(logp)
    plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
    entropy = -plogp.sum(-1)
    tokens = s["tokens"]
    kept = tokens != IGNORE
    at = torch.where(kept, tokens, torch.zeros_like(tokens))[:, None]
    lp = torch.where(kept, logp.gather(1, at)[:, 0], torch.zeros_like(entropy))
    if s["mode"] == "score":
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["top"]]
        return {"logprob": lp, "entropy": entropy, "top_logprobs": logp.gather(1, order), "top_tokens": order}
    gl = (s["dlogprob"] * kept)[:, None]
    gh = s["dentropy"][:, None]
    d = -gl * p - gh * (plogp + p * entropy[:, None])
    d.scatter_add_(1, at, gl * ~empty)
    return {"logprob": lp, "entropy": entropy, "dlogits": d.to(s["logits"].dtype)}


def _run_plain(s):
    kind, mode = s["kind"], s["mode"]
    if kind == "lp":
        return _plain_lp(s)
    x, dt = s["x"].float(), s["x"].dtype
    if mode == "pack":
        return {"x": _read_back(x).to(dt)}
    if mode == "gelu":
        kept = _read_back(x)
        again, slope = _gelu(kept)
        return {"y": _gelu(x)[0].to(dt), "dx": (s["dy"].float() * slope).to(dt), "again": again.to(dt)}
    weight, bias, out = s["weight"], s["bias"], s["out"]
    mean, rstd = _norm_stats(x, s["eps"])
    xhat = (x - mean) * rstd
    r = {"y": (xhat * weight + bias).to(out)}
    if kind == "act8":
        xhat = (_read_back(x) - mean) * rstd
        r["again"] = (xhat * weight + bias).to(out)
    if mode != "forward":
        dx, dw, db = _norm_grads(xhat, rstd, weight, s["dy"].float())
        r.update(dx=dx.to(dt), dweight=dw, dbias=db)
    return r


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    size = _SIZE[c["dtype"]]
    if c["kind"] == "lp":
        n = c["rows"] * c["V"]
        if c["mode"] == "score":
            return {"bytes": n * size + c["rows"] * (16 + 12 * c["top"]), "flops": 6 * n}
        # the logits once in each direction, their gradient written
        return {"bytes": 3 * n * size + 24 * c["rows"], "flops": 14 * n}
    n, rows, D = c["rows"] * c["D"], c["rows"], c["D"]
    kept = n + 4 * rows * -(-D // GROUP)  # a checkpoint's bytes
    if c["mode"] == "pack":
        return {"bytes": 2 * (n * size + kept), "flops": 4 * n}
    if c["mode"] == "gelu":
        # forward: x, y and the checkpoint; backward: dy, the checkpoint, dx and y again
        return {"bytes": 5 * n * size + 2 * kept, "flops": 60 * n}
    osize = _SIZE[c["out"]]
    forward = n * (size + osize) + 8 * D
    if c["mode"] == "forward":
        return {"bytes": forward, "flops": 8 * n}
    back = n * (size + osize) + 8 * rows + 12 * D
    if c["kind"] == "norm":
        # the backward reads x again, dy, and writes dx
        return {"bytes": forward + 8 * rows + back + n * size, "flops": 20 * n}
    # the backward reads the checkpoint and dy and writes dx, and y again before
    return {"bytes": forward + 8 * rows + back + 3 * kept + n * osize, "flops": 32 * n}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_kept(x32):
    """The checkpoint's values by its definition (its scale and steps are float32 by definition), in float64."""
    rows, D = x32.shape
    out = torch.empty(rows, D, dtype=torch.float64, device=x32.device)
    for a in range(0, D, GROUP):
        v = x32[:, a:a + GROUP]
        amax = v.abs().max(1, keepdim=True).values
        q = (v.double() * (127.0 / amax.double()).float().double()).float().round().double()
        out[:, a:a + GROUP] = torch.where(amax < TINY, 0.0, q * (amax.double() * STEP).float().double())
    return out


def _exact_cdf(x):
    return torch.special.erfc(-x / math.sqrt(2.0)) / 2


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "lp":
        parts = []
        step = max(1, (1 << 26) // case["V"])
        for a in range(0, case["rows"], step):  # float64 copies of a part of the rows at a time
            parts.append(_exact_lp(s, slice(a, a + step)))
        return {k: torch.cat([p[k] for p in parts]) if parts[0][k] is not None else None for k in parts[0]}
    x = s["x"].double()
    if case["mode"] == "pack":
        return {"x": _exact_kept(s["x"].float())}
    if case["mode"] == "gelu":
        h = _exact_kept(s["x"].float())
        slope = _exact_cdf(h) + h * torch.exp(-h.square() / 2) / math.sqrt(2 * math.pi)
        return {"y": x * _exact_cdf(x), "dx": s["dy"].double() * slope, "again": h * _exact_cdf(h)}
    w, b = s["weight"].double(), s["bias"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    dev = (var + s["eps"]).sqrt()
    r = {"y": (x - mean) / dev * w + b}
    if case["mode"] == "forward":
        return r
    xh = (x - mean) / dev
    if case["kind"] == "act8":
        xh = (_exact_kept(s["x"].float()) - mean) / dev
        r["again"] = xh * w + b
    dy = s["dy"].double()
    g = dy * w
    D = case["D"]
    r["dx"] = (g - g.sum(1, keepdim=True) / D - xh * ((g * xh).sum(1, keepdim=True) / D)) / dev
    r["dweight"], r["dbias"] = (dy * xh).sum(0), dy.sum(0)
    return r


def _exact_lp(s, part):
    x, tokens = s["logits"][part].double(), s["tokens"][part]
    lse = torch.logsumexp(x, 1, keepdim=True)
    some = torch.isfinite(lse)
    logp = torch.where(some, x - lse, -math.inf)
    p = logp.exp()
    entropy = torch.special.entr(p).sum(1)
    kept = tokens >= 0
    at = tokens.clamp_min(0)[:, None]
    lp = torch.where(kept, logp.gather(1, at)[:, 0], 0.0)
    if s["mode"] == "score":
        rank = torch.argsort(x, dim=1, descending=True, stable=True)[:, :s["top"]]
        return {"logprob": lp, "entropy": entropy, "top_logprobs": logp.gather(1, rank), "top_tokens": rank}
    gl = torch.where(kept, s["dlogprob"][part].double(), 0.0)[:, None]
    gh = s["dentropy"][part].double()[:, None]
    d = gh * (torch.special.entr(p) - p * entropy[:, None]) - gl * p
    hit = torch.zeros_like(p).scatter_(1, at, 1.0)
    return {"logprob": lp, "entropy": entropy, "dlogits": d + gl * hit * some}
