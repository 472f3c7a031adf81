"""Log probabilities from hidden states at sizes where every product is cut into its
largest tiles, over many stages of k, in several pieces of the vocabulary, the last of
them shorter than the others; and of peaked distributions.  Against the formulas in
float64 on the GPU, some rows at a time.

Bounds as in test_gpu_linear_logprobs, in the terms of what the operands' pieces lose:
``SPLIT`` of a type is (what a piece's value is off, relative; what a product of two is
off for the two operands and the products of small pieces that are left out; how many
products a term is).  A weight's gradient sums over all rows, so its bound counts them all
in every part."""
import pytest
import torch

from gmdn_amd import logprobs as lpm
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SUM = 256 * U
B, F = torch.bfloat16, torch.float32
IGNORE = lpm.IGNORE
SPLIT = {B: (2.0 ** -8, 0.0, 1), F: (2.0 ** -16, 3 * 2.0 ** -16, 3)}


def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def data(rows, V, D, dtype, seed, spread=2.0):
    """Inputs on the GPU; a fifth of the tokens are ignored."""
    gen = torch.Generator(device=dev()).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device=dev())

    x, w = rand(rows, D).to(dtype), (rand(V, D) * spread / D ** 0.5).to(dtype)
    tokens = torch.randint(V, (rows,), generator=gen, device=dev())
    tokens[torch.rand(rows, generator=gen, device=dev()) < 0.2] = IGNORE
    return x, w, tokens, rand(rows), 0.1 * rand(rows)


def close(got, ref, tol, what):
    err = (got.double() - ref).abs()
    half = torch.finfo(got.dtype).eps / 2
    bad = ~(err <= tol + half * (ref.abs() + tol) + 1e-38)
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err - tol).max()):.3e}"


def check(x, w, tokens, dl, dh, got, split):
    """got: log probability, entropy, dx, dw of the cotangents dl, dh."""
    lp, entropy, dx, dw = got
    (T, D), V = x.shape, w.shape[0]
    off, pair, products = split
    w64, wa = w.double(), w.double().abs()
    rw, tw = torch.zeros_like(w64), torch.zeros_like(w64)
    for a in range(0, T, 1024):
        part = slice(a, a + 1024)
        x64, at = x[part].double(), tokens[part].clamp(0, V - 1)[:, None]
        l, A = x64 @ w64.t(), x64.abs() @ wa.t()
        top = ((products * (D + 8) * U + pair) * A).amax(1, keepdim=True)
        logp = torch.log_softmax(l, 1)
        size = (l.abs().amax(1) + logp.abs().amax(1)) * 4 * U
        p = logp.exp()
        H = torch.special.entr(p).sum(1)
        kept = tokens[part] != IGNORE
        close(lp[part], torch.where(kept, logp.gather(1, at)[:, 0], 0.0), 2 * top[:, 0] + SUM + size, "lp")
        close(entropy[part], H, 2 * (1 + H) * (top[:, 0] + SUM) + size, "entropy")
        gl, gh = (dl[part] * kept).double()[:, None], dh[part].double()[:, None]
        inner = logp + H[:, None]
        d = (torch.zeros_like(p).scatter_(1, at, 1.0) - p) * gl - gh * p * inner
        td = p * (2 * top + SUM + size[:, None]) * (gl.abs() + gh.abs() * (inner.abs() + 3 + 2 * H[:, None])) + 8 * U * d.abs()
        td += off * (d.abs() + td)
        ad = d.abs() + td
        close(dx[part], d @ w64, td @ wa + (pair + (V + 64) * products * U) * (ad @ wa), "dx")
        rw += d.t() @ x64
        tw += td.t() @ x64.abs() + (pair + (T + 64) * products * U) * (ad.t() @ x64.abs())
    close(dw, rw, tw, "dw")


def run(rows, V, D, dtype, seed, split=None, spread=2.0, **kw):
    x, w, tokens, dl, dh = data(rows, V, D, dtype, seed, spread)
    x.requires_grad_(True), w.requires_grad_(True)
    got = lpm.linear_logprobs(x, w, tokens, **kw)
    grads = torch.autograd.grad(got, [x, w], [dl, dh])
    assert [g.dtype for g in grads] == [dtype] * 2
    check(x.detach(), w.detach(), tokens, dl, dh, [t.detach() for t in (*got, *grads)], split or SPLIT[dtype])


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("rows,V,D", [(1021, 32003, 1001), (2100, 9001, 1024)])
def test_largest_tiles(rows, V, D, dtype):
    """The three products, ragged at every end; dW over 16 and 33 stages, dx over parts of 32
    and 21."""
    run(rows, V, D, dtype, rows + V + D)


@pytest.mark.parametrize("rows,V,D,dtype", [(2049, 65812, 200, F), (8200, 40001, 200, B)])
def test_pieces_of_the_vocabulary(rows, V, D, dtype):
    """Two pieces; in float32 the second has one split of dx less than the first."""
    run(rows, V, D, dtype, rows + V + D)


@pytest.mark.parametrize("dtype", [B, F])
def test_peaked_distributions(dtype):
    """Logits of some hundreds, their gradients too."""
    run(40, 300, 64, dtype, 8, spread=80.0)
