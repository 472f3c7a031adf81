"""GPU parity of log probabilities from hidden states and the head's weight
(csrc/linear_logprobs.hip), forward and backward, against the formulas in
float64.

Bounds, with u = 2^-24 and A = |x| |W|^T, the sums of magnitudes behind the logits.
bfloat16 products are exact in float32 and a logit adds D of them: (D + 8) u A.  float32
operands are two bfloat16 pieces, each rounding off at most 2^-8 of what is left: 2^-16 of
the value, and the product of the two small pieces is left out: 3 2^-16 A in all,
and three times as many sums.  A row's sums of exponentials add up to V / 64 joined
ones; with the exponential's argument (|l - M| below 60 where it counts) they stay
within SUM = 256 u.  Log probability and entropy see the logits' error at most
twice and 2 (1 + H) times.
The logits' gradient d sees it through p, and is rounded to its pieces: 2^-8 |d| in
bfloat16, 2^-16 in float32; the products add V or T terms.  An output adds half a step
of its type."""
import pytest
import torch

from gmdn_amd import logprobs as lpm
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SUM = 256 * U
B, F = torch.bfloat16, torch.float32
IGNORE = lpm.IGNORE


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _data(rows, V, D, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, D, generator=gen).to(dtype)
    w = (torch.randn(V, D, generator=gen) * spread / D ** 0.5).to(dtype)
    tokens = torch.randint(V, (rows,), generator=gen)
    tokens[torch.rand(rows, generator=gen) < 0.2] = IGNORE
    dl, dh = torch.randn(rows, generator=gen), 0.1 * torch.randn(rows, generator=gen)
    return x, w, tokens, dl, dh


def _reference(x, w, tokens, dl, dh):
    """Name -> (value, bound)."""
    f32 = x.dtype == F
    x, w = x.double(), w.double()
    (T, D), V = x.shape, w.shape[0]
    l, A = x @ w.t(), x.abs() @ w.abs().t()
    tl = (3 if f32 else 1) * (D + 8) * U * A + (3 * 2.0 ** -16 * A if f32 else 0)
    top = tl.amax(1, keepdim=True)
    logp = torch.log_softmax(l, 1)
    p, H = logp.exp(), torch.special.entr(logp.exp()).sum(1)
    kept = tokens != IGNORE
    at = tokens.clamp(0, V - 1)[:, None]
    hit = torch.zeros_like(p).scatter_(1, at, 1.0)
    size = (l.abs().amax(1) + logp.abs().amax(1)) * 4 * U
    out = {"lp": (torch.where(kept, logp.gather(1, at)[:, 0], 0.0), 2 * top[:, 0] + SUM + size),
           "entropy": (H, 2 * (1 + H) * (top[:, 0] + SUM) + size)}
    gl, gh = (dl * kept).double()[:, None], dh.double()[:, None]
    d = gl * (hit - p) - gh * p * (logp + H[:, None])
    te = 2 * top + SUM + size[:, None]  # of log p
    td = p * te * (gl.abs() + gh.abs() * ((logp + H[:, None]).abs() + 3 + 2 * H[:, None])) + 8 * U * d.abs()
    td = td + (2.0 ** -16 if f32 else 2.0 ** -8) * (d.abs() + td)
    piece = 2 * 2.0 ** -16 if f32 else 0.0  # of the other operand, and the product left out
    ad = d.abs() + td
    out["dx"] = (d @ w, td @ w.abs() + (piece + (V + 64) * 3 * U) * (ad @ w.abs()))
    out["dw"] = (d.t() @ x, td.t() @ x.abs() + (piece + (T + 64) * 3 * U) * (ad.t() @ x.abs()))
    return out


def _close(got, ref, tol, what):
    err = (got.double().cpu() - ref).abs()
    half = torch.finfo(got.dtype).eps / 2
    bad = ~(err <= tol + half * (ref.abs() + tol) + 1e-38)
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err - tol).max()):.3e}"


def _run(rows, V, D, dtype, seed, use=(True, True), place=lambda t: t):
    dev = _dev()
    x, w, tokens, dl, dh = _data(rows, V, D, dtype, seed)
    xd, wd = (place(t.to(dev, copy=True)).requires_grad_(True) for t in (x, w))
    got = lpm.linear_logprobs(xd, wd, tokens.to(dev))
    assert got.logprob.dtype == got.entropy.dtype == F
    dl, dh = (t if on else torch.zeros_like(t) for t, on in zip((dl, dh), use))
    outs = [t for t, on in zip(got, use) if on]
    dx, dw = torch.autograd.grad(outs, [xd, wd], [t.to(dev) for t, on in zip((dl, dh), use) if on])
    assert dx.dtype == dw.dtype == dtype
    ref = _reference(x, w, tokens, dl, dh)
    for name, t in (("lp", got.logprob), ("entropy", got.entropy), ("dx", dx), ("dw", dw)):
        _close(t.detach(), *ref[name], name)


SIZES = [(1, 1, 1), (1, 2, 3), (3, 5, 7), (8, 300, 64), (2, 65, 128), (70, 70, 70), (64, 64, 64), (65, 129, 192),
         (130, 257, 256), (5, 1000, 40), (200, 33, 100), (1, 700, 64), (1030, 600, 16)]


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("rows,V,D", SIZES)
def test_forward_backward(rows, V, D, dtype):
    _run(rows, V, D, dtype, rows + V + D)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("rows,V,D", [(4001, 4200, 72), (1000, 16500, 64), (4096, 4096, 65), (300, 33000, 128),
                                      (1500, 3001, 200), (257, 2000, 1000), (64, 5000, 40), (2100, 70, 64)])
def test_large_products(rows, V, D, dtype):
    """Sizes at which the products are cut into larger tiles, whole and ragged, and
    split along k."""
    _run(rows, V, D, dtype, rows + V + D)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_one_output_used(use, dtype):
    _run(70, 200, 64, dtype, 1, use)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("which", ["slice", "shifted", "transposed"])
def test_layouts(which, dtype):
    """Rows with a stride, rows off 16-byte addresses, columns of a matrix."""
    def place(t):
        if which == "transposed":
            return t.t().contiguous().t()
        wide = torch.full((t.shape[0], t.shape[1] + 8), float("nan"), dtype=t.dtype, device=t.device)
        at = 8 if which == "slice" else 3
        wide[:, at:at + t.shape[1]] = t
        return wide[:, at:at + t.shape[1]]

    _run(70, 130, 64, dtype, 2, place=place)
    _run(33, 70, 40, dtype, 3, place=place)


def test_batch_and_int32_tokens():
    dev = _dev()
    x, w, tokens, dl, _ = _data(24, 90, 32, B, 4)
    xd, wd = x.view(2, 3, 4, 32).to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    got = lpm.linear_logprobs(xd, wd, tokens.view(2, 3, 4).int().to(dev))
    assert got.logprob.shape == got.entropy.shape == (2, 3, 4)
    dx, dw = torch.autograd.grad(got.logprob, [xd, wd], dl.view(2, 3, 4).to(dev))
    ref = _reference(x, w, tokens, dl, torch.zeros(24))
    _close(got.logprob.detach().view(-1), *ref["lp"], "lp")
    _close(dx.view(24, 32), *ref["dx"], "dx")
    _close(dw, *ref["dw"], "dw")


@pytest.mark.parametrize("need", ["x", "weight"])
def test_one_operand_frozen(need):
    """The other's gradient is the one with nothing frozen, bit for bit."""
    dev = _dev()
    x, w, tokens, dl, _ = _data(70, 300, 64, B, 5)

    def grads(nx, nw):
        xd, wd = x.to(dev, copy=True).requires_grad_(nx), w.to(dev, copy=True).requires_grad_(nw)
        lpm.linear_logprobs(xd, wd, tokens.to(dev)).logprob.backward(dl.to(dev))
        return xd.grad, wd.grad

    whole, some = grads(True, True), grads(need == "x", need == "weight")
    for a, b, wanted in zip(some, whole, (need == "x", need == "weight")):
        assert torch.equal(a, b) if wanted else a is None


def test_tokens_outside_and_ignored():
    """An ignored token: log probability 0, and with no cotangent of the entropy
    no gradient at all; one outside the vocabulary: NaN."""
    dev = _dev()
    x, w, tokens, dl, _ = _data(20, 50, 64, F, 6)
    tokens[:4] = torch.tensor([50, -1, IGNORE, 0])
    xd = x.to(dev).requires_grad_(True)
    got = lpm.linear_logprobs(xd, w.to(dev), tokens.to(dev))
    assert got.logprob[:2].isnan().all() and got.logprob[2] == 0 and got.logprob[3:].isfinite().all()
    assert got.entropy.isfinite().all()
    (dx,) = torch.autograd.grad(got.logprob, xd, dl.to(dev))
    assert dx[:2].isnan().all() and (dx[2] == 0).all() and dx[3:].isfinite().all()
    tokens[:] = IGNORE
    wd = w.to(dev).requires_grad_(True)
    (dw,) = torch.autograd.grad(lpm.linear_logprobs(x.to(dev), wd, tokens.to(dev)).logprob, wd, dl.to(dev))
    assert (dw == 0).all()


def test_nan_stays_in_its_row():
    dev = _dev()
    x, w, tokens, dl, _ = _data(20, 50, 64, B, 7)
    tokens[:] = torch.arange(20)
    x[3, 5] = float("nan")
    xd = x.to(dev).requires_grad_(True)
    got = lpm.linear_logprobs(xd, w.to(dev), tokens.to(dev))
    others = torch.arange(20) != 3
    assert got.logprob[3].isnan() and got.logprob.cpu()[others].isfinite().all()
    (dx,) = torch.autograd.grad(got.logprob, xd, dl.to(dev))
    assert dx[3].isnan().all() and dx.cpu()[others].isfinite().all()


def test_peaked_distributions():
    """Logits of some hundreds: a probability of one, entropy near zero, tails
    below float32."""
    dev = _dev()
    x, w, tokens, dl, dh = _data(40, 300, 64, F, 8, spread=80.0)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    got = lpm.linear_logprobs(xd, wd, tokens.to(dev))
    grads = torch.autograd.grad(got, [xd, wd], [dl.to(dev), dh.to(dev)])
    ref = _reference(x, w, tokens, dl, dh)
    assert all(g.isfinite().all() for g in grads) and (got.entropy >= 0).all()
    _close(got.logprob.detach(), *ref["lp"], "lp")
    _close(got.entropy.detach(), *ref["entropy"], "entropy")


def test_differences():
    """The gradients beside differences of the operator itself."""
    dev = _dev()
    x, w, tokens, dl, dh = _data(4, 30, 16, F, 9)
    leaf = [t.to(dev).requires_grad_(True) for t in (x, w)]

    def value():
        got = lpm.linear_logprobs(*leaf, tokens.to(dev))
        return (got.logprob * dl.to(dev)).double().sum() + (got.entropy * dh.to(dev)).double().sum()

    grads = torch.autograd.grad(value(), leaf)
    h = 2.0 ** -5  # off by h^2 / 6 of a third derivative (below 10 here), and by 3 2^-16 of products below 20 over h
    for t, g in zip(leaf, grads):
        at = t.detach().view(-1)
        for i in range(0, at.numel(), 7):
            keep = at[i].item()
            with torch.no_grad():
                at[i] = keep + h
                up = value()
                at[i] = keep - h
                down = value()
                at[i] = keep
            assert abs(float(up - down) / (2 * h) - float(g.view(-1)[i])) < 0.03


def test_no_rows():
    dev = _dev()
    xd, wd = torch.empty(2, 0, 64, device=dev, requires_grad=True), torch.randn(30, 64).to(dev).requires_grad_(True)
    got = lpm.linear_logprobs(xd, wd, torch.empty(2, 0, dtype=torch.int64, device=dev))
    dx, dw = torch.autograd.grad(got.logprob, [xd, wd], torch.empty(2, 0, device=dev))
    assert got.logprob.shape == (2, 0) and dx.shape == xd.shape and (dw == 0).all()


def test_same_bits_on_every_run():
    dev = _dev()
    x, w, tokens, dl, dh = (t.to(dev) for t in _data(300, 2000, 128, B, 10))

    def call():
        lp, h, stats = torch.ops.gmdn.linear_logprobs_fwd(x, w, tokens, IGNORE)
        return lp, h, *torch.ops.gmdn.linear_logprobs_bwd(x, w, tokens, stats, h, dl, dh, IGNORE, True, True)

    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(call(), first))


def test_cross_entropy():
    """Beside torch's on the logits, with ignored targets."""
    dev = _dev()
    x, w, tokens, _, _ = _data(120, 400, 64, F, 11)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    loss = lpm.linear_cross_entropy(xd, wd, tokens.to(dev))
    dx, dw = torch.autograd.grad(loss, [xd, wd])
    x64, w64 = x.double().requires_grad_(True), w.double().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(x64 @ w64.t(), tokens, ignore_index=IGNORE)
    rx, rw = torch.autograd.grad(want, [x64, w64])
    n = (tokens != IGNORE).sum()
    ref = _reference(x, w, tokens, torch.full((120,), -1.0 / float(n)), torch.zeros(120))
    assert abs(float(loss) - float(want)) <= float(ref["lp"][1].max()) + 8 * U * float(want)
    _close(dx, rx.detach(), ref["dx"][1] + 4 * U * rx.abs(), "dx")
    _close(dw, rw.detach(), ref["dw"][1] + 4 * U * rw.abs(), "dw")


def test_pieces_of_the_vocabulary():
    """A call whose logits' gradient is more than one piece: beside the same
    products by torch in float64 on the GPU."""
    dev = _dev()
    rows, V, D = 16390, 20001, 64
    gen = torch.Generator(device=dev).manual_seed(12)
    x = torch.randn(rows, D, generator=gen, device=dev).to(B)
    w = (torch.randn(V, D, generator=gen, device=dev) * 0.3).to(B)
    tokens = torch.randint(V, (rows,), generator=gen, device=dev)
    dl = torch.randn(rows, generator=gen, device=dev)
    lp, h, stats = torch.ops.gmdn.linear_logprobs_fwd(x, w, tokens, IGNORE)
    dx, dw = torch.ops.gmdn.linear_logprobs_bwd(x, w, tokens, stats, h, dl, None, IGNORE, True, True)
    xd, wd = x.double(), w.double()
    rw, mw = torch.zeros(V, D, dtype=torch.float64, device=dev), torch.zeros(V, D, dtype=torch.float64, device=dev)
    for a in range(0, rows, 2048):
        part = slice(a, a + 2048)
        l = xd[part] @ wd.t()
        logp = torch.log_softmax(l, 1)
        # (D + 8) u A is below 72 u times 40 here
        assert ((lp[part] - logp.gather(1, tokens[part, None])[:, 0]).abs() < 2 * 72 * 40 * U + SUM + 200 * U).all()
        d = -logp.exp() * dl[part, None].double()
        d.scatter_add_(1, tokens[part, None], dl[part, None].double())
        err = d.abs() * (2.0 ** -8 + 2e-3)
        ref, tol = d @ wd, err @ wd.abs()
        assert ((dx[part].double() - ref).abs() <= tol + 2.0 ** -8 * ref.abs() + 1e-7).all()
        rw += d.t() @ xd[part]
        mw += err.t() @ xd[part].abs()
    assert ((dw.double() - rw).abs() <= mw + 2.0 ** -8 * rw.abs() + 1e-7).all()


def test_autocast():
    """Under bfloat16 autocast float32 operands are taken in bfloat16."""
    dev = _dev()
    x, w, tokens, dl, _ = _data(40, 100, 64, F, 13)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    with torch.autocast(dev.type, dtype=B):
        got = lpm.linear_logprobs(xd, wd, tokens.to(dev))
    dx, dw = torch.autograd.grad(got.logprob, [xd, wd], dl.to(dev))
    assert dx.dtype == dw.dtype == F
    ref = _reference(x.to(B), w.to(B), tokens, dl, torch.zeros(40))
    _close(got.logprob.detach(), *ref["lp"], "lp")
    for name, g in (("dx", dx), ("dw", dw)):
        value, tol = ref[name]
        _close(g, value, tol + 2.0 ** -8 * (value.abs() + tol), name)


def test_refusals():
    dev = _dev()
    x, w, tokens = torch.randn(3, 8, device=dev), torch.randn(5, 8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for call, message in [
            (lambda: lpm.linear_logprobs(x.half(), w.half(), tokens), "bfloat16 or float32"),
            (lambda: lpm.linear_logprobs(x, w.bfloat16(), tokens), "of one type"),
            (lambda: lpm.linear_logprobs(x, w[:, :4], tokens), "rows of 4 values"),
            (lambda: lpm.linear_logprobs(x, w[0], tokens), "2 dimensions"),
            (lambda: lpm.linear_logprobs(x, w[:0], tokens), "at least one row"),
            (lambda: lpm.linear_logprobs(x, w, tokens[:2]), "shape"),
            (lambda: lpm.linear_logprobs(x, w, tokens.float()), "int64 or int32"),
            (lambda: lpm.linear_logprobs(x, w.cpu(), tokens), "weight is on")]:
        with pytest.raises(RuntimeError, match=message):
            call()
