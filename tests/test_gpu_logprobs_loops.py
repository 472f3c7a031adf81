"""GPU parity of the log probabilities' forward and plain gradient in rows
long enough for the loops over four pieces at a time, in each shape of
workgroup, against float64.

Shapes: 16 threads a row up to 512 logits, 64 up to 4096, then 256 in the
forward (over 1 part, or parts where rows are few) and 256 up to 8192 or 1024 in
the gradient.  The loop over four pieces wants a span of 24 threads + 8.

Bounds, u = 2^-24.  A thread adds n = span / threads + 8 terms, each within 4 u,
and rescales its sum at most once for each eight of them (an exponential and a
product, 5 u); ten joins more.  So the sum is within DELTA = (2 n + 32) u
relative, and its logarithm as much absolute.  log p = x - m - logs adds a
rounding of each step; p, an exponential of it whose argument is scaled and
halved, 2 u |log p| + 10 u; the entropy DELTA of each of its terms; the
gradient one rounding a product."""
import math

import pytest
import torch

from gmdn_amd import logprobs as lp
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SIZES = [(40, 509), (40, 4093), (20, 8189), (300, 24600), (300, 32003), (200, 52001), (1, 90001)]


def _threads(V):
    return 16 if V <= 512 else 64 if V <= 4096 else 256 if V <= 8192 else 1024


def _case(rows, V, dtype):
    """Tokens in each of the four pieces a thread takes at a time, at both ends
    of a piece and of the threads, in the remainder, and in the row's last
    logit; one ignored; a row masked to three logits with its token masked, one
    masked to half, one without any."""
    gen = torch.Generator().manual_seed(rows + V)
    x = 3 * torch.randn(rows, V, generator=gen)
    t = _threads(V)
    at = [V - 1, 0] + [8 * t * i + 8 * k + j for i in range(4) for k in (0, t - 1) for j in (0, 7)]
    at = [a for a in at if a < V] + [V - 2, V - 8, V // 2]
    tokens = torch.tensor([at[r % len(at)] for r in range(rows)])
    if rows > 4:
        tokens[1] = lp.IGNORE
        keep = x[2, [7, V // 2, V - 1]].clone()
        x[2] = -math.inf
        x[2, [7, V // 2, V - 1]] = keep
        x[3, ::2] = -math.inf
        x[4] = -math.inf
    cot = [torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)]
    return x.to(dtype), tokens, cot


def _reference(x, tokens, cot):
    V = x.shape[1]
    n = V / (16 if V <= 512 else 64 if V <= 4096 else 256) + 8
    delta = (2 * n + 32) * U
    x = x.double()
    m = x.amax(1, keepdim=True)
    some = m > -math.inf
    m = torch.where(some, m, 0.0)
    logs = torch.where(some, torch.exp(x - m).sum(1, keepdim=True).log(), 0.0)
    logp = torch.where(some, x - m - logs, -math.inf)
    p = logp.exp()
    size = torch.where(p == 0, 0.0, logp).abs()
    H = (p * size).sum(1, keepdim=True)
    dl = delta + U * ((x - m).nan_to_num(neginf=0.0).abs() + size + 3 * logs)
    dH = delta * (logs + 2 * H + 4)
    kept = tokens != lp.IGNORE
    at = torch.where(kept, tokens, 0)[:, None]
    gl, gh = (c.double()[:, None] for c in cot)
    gl = torch.where(kept[:, None], gl, 0.0)
    d = -p * (gl + gh * (H - size))
    err = p * ((dl + U * (2 * size + 10)) * (gl.abs() + gh.abs() * (size + H))
               + gh.abs() * (dl + dH + 2 * U * (size + H)) + 2 * U * gl.abs())
    hit = torch.zeros_like(p).scatter_(1, at, 1.0) * some
    lg = torch.where(kept, logp.gather(1, at)[:, 0], 0.0)
    return ((lg, torch.where(kept, dl.gather(1, at)[:, 0], 0.0)), (H[:, 0], dH[:, 0]),
            (d + hit * gl, err + hit * 4 * U * gl.abs()))


def _close(got, ref, tol, what):
    bits = 8 if got.dtype == torch.bfloat16 else 24
    got = got.detach().double().cpu()
    half = torch.pow(2.0, torch.floor(torch.log2(ref.abs().clamp_min(1e-300))) - bits) * (1 + 2 ** -6) + 2.0 ** -126
    same = got == ref  # the infinities
    bad = ~(same | ((got - ref).abs() <= tol + half))
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V", SIZES)
def test_plain_gradient_of_long_rows(rows, V, dtype):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    x, tokens, cot = _case(rows, V, dtype)
    leaf = x.cuda().requires_grad_(True)
    got = lp.token_logprobs(leaf, tokens.cuda())
    (d,) = torch.autograd.grad(got[:2], leaf, [c.cuda() for c in cot])
    logprob, entropy, grad = _reference(x, tokens, cot)
    _close(got.logprob, *logprob, "logprob")
    _close(got.entropy, *entropy, "entropy")
    _close(d, *grad, "dlogits")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V", [(40, 509), (40, 4093), (20, 8189), (300, 32003)])
def test_every_column_has_its_token_term(rows, V, dtype):
    """The token's term by itself: with the cotangent of the log probability 1
    and logits that are all equal, a gradient is 1 - 1/V at the token and -1/V
    elsewhere, whichever column the token is (each of them for the short rows,
    a stride of them for the long)."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    x = torch.zeros(rows, V, dtype=dtype, device="cuda").requires_grad_(True)
    step = max(1, V // 1500) | 1
    columns = torch.arange(0, V, step, device="cuda")
    for part in columns.split(rows):
        tokens = torch.cat([part, part.new_full((rows - len(part),), V - 1)])
        (d,) = torch.autograd.grad(lp.token_logprobs(x, tokens).logprob.sum(), x)
        want = torch.full((rows, V), -1.0 / V, dtype=torch.float64, device="cuda")
        want.scatter_(1, tokens[:, None], 1 - 1.0 / V)
        eps = 2.0 ** -8 if dtype == torch.bfloat16 else (4 * (V / 16 + 8) + 64) * U
        assert ((d.double() - want).abs() <= want.abs() * eps).all()
