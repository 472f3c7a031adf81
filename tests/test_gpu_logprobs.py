"""GPU parity of the token log probabilities (csrc/logprobs.hip): log
probability, entropy, top alternatives and the logits' gradient, against
float64.

Bounds, with u = 2^-24: a thread adds at most V / 2048 + 32 terms in sequence
and the row's sum joins ten levels, each term's exponential within 4 u; so the
sum's relative error is below DELTA = (V / 2048 + 64) u, which is the absolute
error of its logarithm; a difference of logits adds u of itself."""
import math

import pytest
import torch
import torch.nn.functional as F

from gmdn_amd import logprobs as lp
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float32]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def delta(V):
    return (V / 2048 + 64) * U


def reference(x, tokens, top, cot=None):
    """Values and, for cotangents (of logprob, entropy, alternatives), the
    gradient, in float64, each with its bound."""
    x = x.double()
    V = x.shape[-1]
    peak = x.amax(-1, keepdim=True)
    empty = peak == -math.inf
    base = torch.where(empty, 0.0, peak)
    logs = torch.log(torch.exp(x - base).sum(-1, keepdim=True))
    logp = torch.where(empty, -math.inf, x - base - logs)
    p = logp.exp()
    plogp = torch.where(p == 0, 0.0, p * logp)
    H = -plogp.sum(-1)
    size = torch.where(empty, 0.0, logs)
    tol = delta(V) + 4 * U * (torch.where(p == 0, 0.0, logp).abs() + 2 * size.abs())
    kept = tokens != lp.IGNORE
    at = torch.where(kept, tokens, 0)[..., None]
    order = torch.argsort(x, dim=-1, descending=True, stable=True)[..., :top]
    tol_h = delta(V) * (size[..., 0] + 2 * H + 4)
    out = {"logprob": (torch.where(kept, logp.gather(-1, at)[..., 0], 0.0), tol.gather(-1, at)[..., 0]),
           "entropy": (H, tol_h), "top_logprobs": (logp.gather(-1, order), tol.gather(-1, order)), "top_tokens": order}
    if cot is not None:
        gl, gh, gt = (c.double() for c in cot)
        gl = torch.where(kept, gl, 0.0)[..., None]
        gh = gh[..., None]
        G = gl + gt.sum(-1, keepdim=True)
        hit = torch.zeros_like(p).scatter_add_(-1, at, gl).scatter_add_(-1, order, gt) * ~empty
        mag = gl.abs() + gt.abs().sum(-1, keepdim=True)
        d = hit - G * p - gh * (plogp + p * H[..., None])
        rel = tol + U * (8 + 4 * torch.where(p == 0, 0.0, logp).abs())
        bound = (p * rel * (mag + gh.abs() * (torch.where(p == 0, 0.0, logp).abs() + H[..., None] + 1))
                 + p * gh.abs() * tol_h[..., None] + U * 40 * mag * (hit != 0) + U * 40 * mag * p)
        out["dlogits"] = (d, bound)
    return out


def assert_close(got, ref, tol, what):
    got = got.double().cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine), what
    assert torch.equal(got[~fine].nan_to_num(nan=7.0), ref[~fine].nan_to_num(nan=7.0)), what
    err = (got - ref).abs()[fine]
    bad = ~(err <= tol[fine])
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err - tol[fine]).max()):.3e}"


def half(ref, dtype):
    bits = 8 if dtype == torch.bfloat16 else 24
    return torch.pow(2.0, torch.floor(torch.log2(ref.abs().clamp_min(1e-300))) - bits) * (1 + 2 ** -6) + 2.0 ** -126


def check(x, tokens, top, seed=0, ignore=True):
    """Values and gradients of CPU logits and tokens against the reference."""
    dev = _dev()
    gen = torch.Generator().manual_seed(seed)
    cot = [torch.randn(tokens.shape, generator=gen), torch.randn(tokens.shape, generator=gen),
           torch.randn((*tokens.shape, top), generator=gen)]
    ref = reference(x, tokens, top, cot)
    xd = x.to(dev).requires_grad_(True)
    got = lp.token_logprobs(xd, tokens.to(dev), top)
    assert got.logprob.dtype == got.entropy.dtype == got.top_logprobs.dtype == torch.float32
    for name in ("logprob", "entropy", "top_logprobs"):
        r, t = ref[name]
        assert_close(getattr(got, name).detach(), r, t + U * r.abs().nan_to_num(posinf=0.0), name)
    assert torch.equal(got.top_tokens.cpu(), ref["top_tokens"])
    (d,) = torch.autograd.grad(got[:3] if top else got[:2], xd, [c.to(dev) for c in (cot if top else cot[:2])])
    assert d.dtype == x.dtype and d.shape == x.shape
    r, t = ref["dlogits"]
    assert_close(d, r, t + half(r, x.dtype), "dlogits")


def logits(shape, seed, dtype, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(shape, generator=gen)
    tokens = torch.randint(shape[-1], shape[:-1], generator=gen)
    if tokens.numel() > 2:
        tokens.view(-1)[1] = lp.IGNORE
    return x.to(dtype), tokens


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (3, 2, 2), (4, 7, 3), (5, 8, 8), (3, 64, 32), (4, 65, 5),
                                        (9, 257, 20), (300, 1000, 0), (5, 4099, 32), (3, 8192, 20), (3, 8193, 20),
                                        (4, 32000, 20), (2, 32768, 32), (2, 32769, 7), (2, 70001, 20), (2, 131072, 0),
                                        (1, 300001, 32), (1, 600000, 32)])
def test_values_and_gradient(rows, V, top, dtype):
    check(*logits((rows, V), V + rows, dtype), top)


@pytest.mark.parametrize("dtype", TYPES)
def test_leading_dimensions_and_strides(dtype):
    """(B, T, V) logits, a padded vocabulary's slice at an odd offset, a
    transposed batch and int32 tokens give what contiguous copies give."""
    dev = _dev()
    wide, tokens = logits((3, 5, 531), 4, dtype)
    wide, tokens = wide.to(dev), tokens.to(dev) % 500
    for x, t in ((wide, tokens), (wide[..., 3:503], tokens), (wide[..., :517], tokens.int()),
                 (wide.transpose(0, 1), tokens.t()), (wide[:, 1:2].expand(3, 5, 531), tokens), (wide[0, 0], tokens[0, 0])):
        got = lp.token_logprobs(x, t, 4)
        want = lp.token_logprobs(x.contiguous(), t.contiguous().long(), 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert got.logprob.shape == t.shape and got.top_tokens.shape == (*t.shape, 4)
    assert lp.token_logprobs(wide[:0], tokens[:0], 3).top_tokens.shape == (0, 5, 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [100, 9000, 40000])
def test_masks(V, dtype):
    """-inf logits: rows with a few tokens left, with fewer than asked for, with
    one, with none, the given token masked; the last pieces only; and masks of
    the type's lowest value, which are a logit like others."""
    x, tokens = logits((9, V), V, dtype)
    gen = torch.Generator().manual_seed(1)
    x[0, torch.rand(V, generator=gen) < 0.9] = -math.inf
    keep = x[1, [5, V // 2, V - 1]].clone()
    x[1] = -math.inf
    x[1, [5, V // 2, V - 1]] = keep
    x[2] = -math.inf
    x[2, V - 1] = -4.0
    x[3] = -math.inf
    x[4, tokens[4]] = -math.inf
    x[5, :V - 3] = -math.inf
    x[6] = torch.finfo(dtype).min
    x[7, 1:] = torch.finfo(dtype).min
    tokens[3], tokens[7] = 11, 0
    check(x, tokens, 20)
    check(x, tokens, 0)


@pytest.mark.parametrize("mask", [-math.inf, -1e30, -3.0])
@pytest.mark.parametrize("rows,V", [(24, 600), (1030, 1220), (24, 7681), (24, 20000), (260, 9001), (3, 140000)])
def test_handfuls(rows, V, mask):
    """Rows with 0 to 40 logits beside the masks, one piece of them, and one in
    each of the first columns' pieces."""
    gen = torch.Generator().manual_seed(V)
    x = torch.full((rows, V), mask)
    for r in range(min(rows, 24)):
        at = torch.randperm(V, generator=gen)[:2 * r if r < 21 else 8]
        at = at if r < 21 else torch.arange(8) + 16 if r == 21 else 8 * torch.arange(8) + r
        x[r, at] = torch.randn(len(at), generator=gen)
    x[24:] = x[:24].repeat(rows // 24 + 1, 1)[24:rows]
    tokens = torch.randint(V, (rows,), generator=gen)
    for top in (1, 8, 32):
        check(x, tokens, top)


@pytest.mark.parametrize("V", [600, 20000, 50000, 150000])
def test_ties_and_orders(V):
    """Equal logits go by index, whatever their number; rising, falling and
    blockwise rows; a row whose likely tokens crowd a few groups (more
    candidates than the list holds: the row is done over)."""
    gen = torch.Generator().manual_seed(2)
    x = torch.zeros(8, V)
    x[1] = torch.arange(V).float() / V
    x[2] = -torch.arange(V).float() / V
    x[3] = torch.randint(3, (V,), generator=gen).float()
    x[4] = (torch.arange(V) // 512).float()
    x[5] = torch.where((torch.arange(V) // 8) % 64 < 31, 5.0 + torch.rand(V, generator=gen), torch.rand(V, generator=gen))
    x[6] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    x[7, V - 40:] = 1.0
    tokens = torch.randint(V, (8,), generator=gen)
    for top in (1, 20, 32):
        check(x, tokens, top)
        check(x.bfloat16(), tokens, top)


@pytest.mark.parametrize("rows,V,top", [(300, 9001, 5), (300, 40000, 32), (700, 300, 0), (300, 5000, 20),
                                        (1100, 257, 20), (1030, 2047, 32), (1024, 8, 8)])
def test_many_rows(rows, V, top):
    """Row counts that take other shapes of workgroup than a few rows do."""
    check(*logits((rows, V), rows + V, torch.bfloat16), top)


def test_ties_in_many_short_rows():
    """Equal logits, sorted rows and masks where a row is one wave's."""
    V, gen = 1500, torch.Generator().manual_seed(7)
    x = torch.randn(1200, V, generator=gen)
    x[::7] = 0.0
    x[1::7] = torch.arange(V).float()
    x[2::7] = -torch.arange(V).float()
    x[3::7, 9:] = -math.inf
    x[4::7] = torch.randint(2, (172, V), generator=gen).float()[:x[4::7].shape[0]]
    x[5::7] = torch.where((torch.arange(V) // 8) % 64 < 31, 1.0 + torch.rand(V, generator=gen), 0.0)
    x[6] = -math.inf
    tokens = torch.randint(V, (1200,), generator=gen)
    for top in (1, 20, 32):
        check(x, tokens, top)


def test_large_matrices_equal_their_parts():
    """Beyond 96 MB logits are loaded past the caches: the same bits."""
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(4)
    x = (3 * torch.randn(1700, 32000, generator=gen, device=dev)).bfloat16()
    tokens = torch.randint(32000, (1700,), generator=gen, device=dev)
    got = lp.token_logprobs(x, tokens)
    for a in (0, 1500):
        part = lp.token_logprobs(x[a:a + 200], tokens[a:a + 200])
        assert torch.equal(got.logprob[a:a + 200], part.logprob) and torch.equal(got.entropy[a:a + 200], part.entropy)


@pytest.mark.parametrize("top", [0, 2])
def test_many_short_rows(top):
    """More rows than a launch has threads for, a workgroup a row: the bits of
    their parts."""
    dev = _dev()
    rows, V = (1 << 24) + 5, 5
    gen = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn(rows, V, generator=gen, device=dev).bfloat16()
    tokens = torch.randint(V, (rows,), generator=gen, device=dev)
    g = torch.randn(rows, generator=gen, device=dev)

    def run(a, b):
        out = torch.ops.gmdn.logprobs_fwd(x[a:b], tokens[a:b], top, -100)
        dtop = g[a:b, None].expand(b - a, top).contiguous() if top else None
        return (*out, torch.ops.gmdn.logprobs_bwd(x[a:b], tokens[a:b], out[4], out[1], out[3], g[a:b], None, dtop, -100))

    got = run(0, rows)
    for a in (0, (1 << 21) - 700, (1 << 23) - 700, rows - 1500):
        for whole, part in zip(got, run(a, a + 1500)):
            assert torch.equal(whole[a:a + 1500], part)


def test_large_and_peaked_logits():
    """Logits far from zero, and a token with nearly all the probability: its
    log probability keeps relative accuracy to float32's resolution of 1."""
    x, tokens = logits((6, 3001), 3, torch.float32, 20.0)
    x[1] += 1e4
    x[2] -= 1e4
    x[3, 17] = 60.0 + x[3].max()
    tokens[3] = 17
    check(x, tokens, 8)


def test_nonfinite_rows():
    """A NaN or +inf makes its own row NaN, and its alternatives go NaN first,
    then by value; other rows are untouched."""
    dev = _dev()
    x, tokens = logits((5, 5000), 8, torch.float32)
    x[1, 0] = math.nan
    x[1, 4000] = math.nan
    x[3, 77] = math.inf
    got = lp.token_logprobs(x.to(dev), tokens.to(dev), 5)
    assert got.entropy[[1, 3]].isnan().all() and got.top_logprobs[[1, 3]].isnan().all()
    want = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :5]
    assert torch.equal(got.top_tokens.cpu(), want)
    ok = [0, 2, 4]
    alone = lp.token_logprobs(x[ok].to(dev), tokens[ok].to(dev), 5)
    assert torch.equal(got.top_logprobs[ok], alone.top_logprobs) and torch.isfinite(alone.top_logprobs).all()
    xd = x.to(dev).requires_grad_(True)
    (d,) = torch.autograd.grad(lp.token_logprobs(xd, tokens.to(dev)).entropy.sum(), xd)
    assert d[[1, 3]].isnan().all() and torch.isfinite(d[ok]).all()


def test_tokens_outside_the_vocabulary():
    """NaN for the position and its gradient, nothing read elsewhere; an
    ignored position has log probability 0, its entropy, and the entropy's
    gradient only."""
    dev = _dev()
    x, _ = logits((4, 50), 1, torch.float32)
    tokens = torch.tensor([50, -1, lp.IGNORE, 3])
    xd = x.to(dev).requires_grad_(True)
    got = lp.token_logprobs(xd, tokens.to(dev), 2)
    assert got.logprob.isnan().tolist() == [True, True, False, False] and got.logprob[2] == 0
    assert torch.isfinite(got.entropy).all()
    (d,) = torch.autograd.grad(got.logprob.sum(), xd)
    assert d[:2].isnan().all() and d[2].eq(0).all() and d[3].ne(0).any()
    assert torch.equal(lp.token_logprobs(xd, torch.full_like(tokens, 7).to(dev), ignore_index=7).logprob,
                       torch.zeros(4, device=dev))


def test_alternatives_and_token_share_a_gradient():
    """The given token among the alternatives, with cotangents on both."""
    dev = _dev()
    x, _ = logits((3, 400), 5, torch.float32)
    tokens = x.argmax(-1)
    check(x, tokens, 6)
    xd = x.to(dev).requires_grad_(True)
    got = lp.token_logprobs(xd, tokens.to(dev), 1)
    a = torch.autograd.grad(got.logprob.sum(), xd, retain_graph=True)[0]
    b = torch.autograd.grad(got.top_logprobs.sum(), xd)[0]
    assert torch.equal(a, b)


def test_gradient_against_differences():
    """Directional derivatives by central differences of the operator's own
    forward at two steps: their difference bounds the truncation, and the
    values' bounds the rounding."""
    dev = _dev()
    x, tokens = logits((3, 90), 12, torch.float32, 1.0)
    gen = torch.Generator().manual_seed(3)
    x, tokens = x.to(dev), tokens.to(dev)
    v = torch.randn(x.shape, generator=gen).to(dev)
    for pick in range(3):
        xd = x.clone().requires_grad_(True)
        (d,) = torch.autograd.grad(lp.token_logprobs(xd, tokens, 4)[pick].sum(), xd)

        def slope(h):
            p, m = (lp.token_logprobs(x + s * h * v, tokens, 4)[pick].double().sum().item() for s in (1, -1))
            return (p - m) / (2 * h)

        d1, d2 = slope(0.01), slope(0.02)
        got = (d.double() * v.double()).sum().item()
        assert abs(got - d1) <= abs(d2 - d1) + 12 * (delta(90) + 16 * U) * 4 / 0.01, (pick, got, d1, d2)


def test_rows_beyond_32_bit_offsets():
    """Rows whose elements lie past 2^31 elements and 2^32 bytes."""
    dev = _dev()
    stride = (1 << 30) + 64
    V = 4097
    base = torch.empty(2 * stride + V, dtype=torch.bfloat16, device=dev)
    x = base.as_strided((3, V), (stride, 1))
    small, tokens = logits((3, V), 6, torch.bfloat16)
    x.copy_(small)
    got = lp.token_logprobs(x, tokens.to(dev), 9)
    want = lp.token_logprobs(small.to(dev), tokens.to(dev), 9)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("ignored", [False, True])
def test_cross_entropy(ignored):
    """The LM's loss and its gradient beside torch's on the float32 logits."""
    dev = _dev()
    x, targets = logits((2, 300, 1000), 2, torch.bfloat16)
    targets = targets.clamp_min(0)
    if ignored:
        targets[0, 100:] = lp.IGNORE
    xd = x.to(dev).requires_grad_(True)
    loss = lp.cross_entropy(xd, targets.to(dev))
    (d,) = torch.autograd.grad(loss, xd)
    x64 = x.double().requires_grad_(True)
    ref = F.cross_entropy(x64.view(-1, 1000), targets.view(-1))
    (r,) = torch.autograd.grad(ref, x64)
    assert abs(loss.item() - ref.item()) <= (delta(1000) + 64 * U) * (1 + abs(ref.item()))
    n = int((targets != lp.IGNORE).sum())
    assert ((d.double().cpu() - r).abs() <= half(r, torch.bfloat16) + 4 * delta(1000) * (r.abs() + 1e-6 / n)).all()


def test_deterministic_and_on_another_stream():
    dev = _dev()
    x, tokens = logits((300, 20001), 1, torch.bfloat16)
    x, tokens = x.to(dev).requires_grad_(True), tokens.to(dev)

    def once():
        got = lp.token_logprobs(x, tokens, 20)
        return (*got, torch.autograd.grad(got.logprob.sum() + got.entropy.sum(), x)[0])

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals():
    dev = _dev()
    x, tokens = logits((4, 40), 1, torch.float32)
    x, tokens = x.to(dev), tokens.to(dev)
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        lp.token_logprobs(x.half(), tokens)
    with pytest.raises(RuntimeError, match="top is"):
        lp.token_logprobs(x, tokens, 33)
    with pytest.raises(RuntimeError, match="top is"):
        lp.token_logprobs(x[:, :5], tokens, 6)
    with pytest.raises(RuntimeError, match="top is"):
        lp.token_logprobs(x, tokens, -1)
    with pytest.raises(RuntimeError, match="tokens has shape"):
        lp.token_logprobs(x, tokens[:3])
    with pytest.raises(RuntimeError, match="tokens are"):
        lp.token_logprobs(x, tokens.float())
    with pytest.raises(RuntimeError, match="tokens is on"):
        lp.token_logprobs(x, tokens.cpu())
    with pytest.raises(RuntimeError, match="at least one value"):
        lp.token_logprobs(x[:, :0], tokens)
    _, h, _, top, stats = torch.ops.gmdn.logprobs_fwd(x, tokens, 2, lp.IGNORE)
    with pytest.raises(RuntimeError, match="stats has shape"):
        torch.ops.gmdn.logprobs_bwd(x, tokens, stats[:, :1], h, top, None, h, None, lp.IGNORE)
    with pytest.raises(RuntimeError, match="dtop has shape"):
        torch.ops.gmdn.logprobs_bwd(x, tokens, stats, h, top, None, None, h, lp.IGNORE)
