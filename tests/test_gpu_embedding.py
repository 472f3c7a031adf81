"""GPU parity of the token embedding and its gradient (csrc/embed.hip).

The forward is one product rounded once: equal bit for bit.  A row of the
gradient is a sum of n rows in float32, in some order: with u = 2^-24 it is within
(n + 2) u of the sum of magnitudes (one more for the scale), and half a step of the
gradient's type from there."""
import pytest
import torch

from gmdn_amd import embedding as em
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float32]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _check_grad(got, tokens, dy, vocab, scale, padding_idx=None):
    tokens, dy = tokens.reshape(-1).long(), dy.reshape(-1, dy.shape[-1]).double() * scale
    keep = (tokens >= 0) & (tokens < vocab) & (tokens != (-1 if padding_idx is None else padding_idx))
    ref = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    mag, n = ref.clone(), torch.zeros(vocab, 1, dtype=torch.float64)
    ref.index_add_(0, tokens[keep], dy[keep])
    mag.index_add_(0, tokens[keep], dy[keep].abs())
    n.index_add_(0, tokens[keep], torch.ones(int(keep.sum()), 1, dtype=torch.float64))
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double().cpu() - ref).abs()
    assert (err <= half * ref.abs() * (1 + 2 ** -6) + (n + 2) * U * mag + 1e-38).all(), float(err.max())
    assert (got.cpu()[n[:, 0] == 0] == 0).all()


def _data(rows, vocab, d, dtype, seed, shape=None):
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(vocab, d, generator=gen).to(dtype)
    # frequent and rare tokens
    tokens = ((vocab + 1.0) ** torch.rand(rows, generator=gen) - 1).long().clamp_(0, vocab - 1)
    dy = torch.randn(rows, d, generator=gen).to(dtype)
    return w, tokens, dy


SIZES = [(1, 1, 1), (1, 7, 5), (5, 3, 8), (33, 10, 16), (64, 100, 64), (65, 513, 65), (300, 17, 24), (1025, 70, 9),
         (2500, 40, 130), (129, 300, 1001), (70, 66, 2050), (40, 9, 4100), (4099, 1003, 200), (300, 70000, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,d", SIZES)
def test_forward_backward(rows, vocab, d, dtype):
    dev = _dev()
    w, tokens, dy = _data(rows, vocab, d, dtype, rows + d)
    wd = w.to(dev, copy=True).requires_grad_(True)
    for scale in (1.0, 3.7):
        y = em.embedding(tokens.to(dev), wd, scale)
        want = (w.float()[tokens] * torch.tensor(scale, dtype=torch.float32)).to(dtype)
        assert y.dtype == dtype and torch.equal(y.detach().cpu(), want)
        (dw,) = torch.autograd.grad(y, wd, dy.to(dev))
        _check_grad(dw, tokens, dy, vocab, scale)


@pytest.mark.parametrize("rows", [32768, 32769, 70000, 300000])
def test_many_tokens(rows):
    """Past the sizes at which each workgroup counts all digits itself, and past
    one tile of the sort each."""
    dev = _dev()
    w, tokens, dy = _data(rows, 5003, 8, torch.float32, rows)
    got = torch.ops.gmdn.embed_bwd(dy.to(dev), tokens.to(dev), 5003, 1.0, -1)
    _check_grad(got, tokens, dy, 5003, 1.0)


@pytest.mark.parametrize("vocab", [511, 512, 513, 262143, 262144, 300000])
def test_digits(vocab):
    """One, two and three passes over the digits, at their borders."""
    dev = _dev()
    gen = torch.Generator().manual_seed(vocab)
    tokens = torch.randint(vocab, (700,), generator=gen)
    tokens[:3] = torch.tensor([vocab - 1, 0, vocab - 1])
    dy = torch.randn(700, 4, generator=gen)
    got = torch.ops.gmdn.embed_bwd(dy.to(dev), tokens.to(dev), vocab, 1.0, -1)
    _check_grad(got, tokens, dy, vocab, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 64, 1000, 40000])
def test_one_token(rows, dtype):
    """All positions one token: its run crosses every block of the sums."""
    dev = _dev()
    dy = torch.randn(rows, 40, generator=torch.Generator().manual_seed(rows)).to(dtype)
    tokens = torch.full((rows,), 3)
    got = torch.ops.gmdn.embed_bwd(dy.to(dev), tokens.to(dev), 5, 0.5, -1)
    _check_grad(got, tokens, dy, 5, 0.5)


def test_padding_and_tokens_outside():
    """The padding row is looked up and gets no gradient; a token outside the
    table gives NaN and none."""
    dev = _dev()
    w, tokens, dy = _data(200, 30, 24, torch.float32, 0)
    tokens[::3] = 29
    for padding_idx in (29, -1):
        wd = w.to(dev, copy=True).requires_grad_(True)
        y = em.embedding(tokens.to(dev), wd, 1.0, padding_idx)
        assert torch.equal(y.detach().cpu(), w[tokens])
        y.backward(dy.to(dev))
        _check_grad(wd.grad, tokens, dy, 30, 1.0, 29)
    tokens[5], tokens[6], tokens[7] = 30, -1, -(1 << 40)
    wd = w.to(dev, copy=True).requires_grad_(True)
    y = em.embedding(tokens.to(dev), wd)
    assert y[5:8].isnan().all() and torch.equal(y[8:].detach().cpu(), w[tokens[8:]])
    y.backward(dy.to(dev))
    _check_grad(wd.grad, tokens, dy, 30, 1.0)


def test_layouts():
    """Batches of tokens in 32 bits, a table that is a slice of a wider one, a
    broadcast cotangent, a transposed one."""
    dev = _dev()
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(50, 99, generator=gen)
    tokens = torch.randint(50, (3, 7), generator=gen, dtype=torch.int32)
    w = wide.to(dev)[:, 1:98].requires_grad_(True)
    y = em.embedding(tokens.to(dev), w)
    assert y.shape == (3, 7, 97) and torch.equal(y.detach().cpu(), wide[:, 1:98][tokens.long()])
    dy = torch.randn(97, generator=gen)
    (dw,) = torch.autograd.grad(y, w, dy.to(dev).expand(3, 7, 97), retain_graph=True)
    _check_grad(dw, tokens, dy.expand(3, 7, 97), 50, 1.0)
    dy = torch.randn(7, 3, 97, generator=gen)
    (dw,) = torch.autograd.grad(y, w, dy.to(dev).transpose(0, 1))
    _check_grad(dw, tokens, dy.transpose(0, 1), 50, 1.0)


def test_no_tokens():
    dev = _dev()
    w = torch.randn(5, 8).to(dev).requires_grad_(True)
    y = em.embedding(torch.empty(2, 0, dtype=torch.int64, device=dev), w)
    assert y.shape == (2, 0, 8)
    (dw,) = torch.autograd.grad(y, w, torch.empty_like(y))
    assert (dw == 0).all() and dw.shape == w.shape


def test_same_bits_on_every_run():
    dev = _dev()
    _, tokens, dy = _data(5000, 300, 72, torch.float32, 4)
    tokens, dy = tokens.to(dev), dy.to(dev)
    first = torch.ops.gmdn.embed_bwd(dy, tokens, 300, 1.0, -1)
    for _ in range(3):
        assert torch.equal(torch.ops.gmdn.embed_bwd(dy, tokens, 300, 1.0, -1), first)


def test_module():
    """The module beside nn.Embedding: parameters, padding, gradients."""
    dev = _dev()
    torch.manual_seed(0)
    ours, theirs = em.Embedding(40, 16, padding_idx=-3, scale=2.0), torch.nn.Embedding(40, 16, padding_idx=-3)
    theirs.load_state_dict(ours.state_dict())
    ours, theirs = ours.to(dev), theirs.to(dev)
    tokens = torch.randint(40, (6, 9), generator=torch.Generator().manual_seed(2)).to(dev)
    tokens[0] = 37
    a, b = ours(tokens), 2.0 * theirs(tokens)
    assert torch.equal(a, b)
    dy = torch.randn(a.shape, generator=torch.Generator().manual_seed(3)).to(dev)
    a.backward(dy)
    b.backward(dy)
    assert torch.allclose(ours.weight.grad, theirs.weight.grad, rtol=1e-5, atol=1e-5)
    assert (ours.weight.grad[37] == 0).all()


def test_refusals():
    dev = _dev()
    w, tokens = torch.randn(5, 8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    dy = torch.randn(3, 8, device=dev)
    op = torch.ops.gmdn
    for call, message in [
            (lambda: em.embedding(tokens, w.half()), "bfloat16 or float32"),
            (lambda: em.embedding(tokens.float(), w), "int64 or int32"),
            (lambda: em.embedding(tokens, w[0]), "2 dimensions"),
            (lambda: em.embedding(tokens, w[:0]), "at least one row"),
            (lambda: em.embedding(tokens.cpu(), w), "tokens is on"),
            (lambda: op.embed_bwd(dy, tokens[:2], 5, 1.0, -1), "shape"),
            (lambda: op.embed_bwd(dy, tokens, 0, 1.0, -1), "at least one row"),
            (lambda: op.embed_bwd(dy, tokens, (1 << 27) + 1, 1.0, -1), "failed with code")]:
        with pytest.raises((RuntimeError, IndexError), match=message):
            call()
    with pytest.raises(ValueError, match="outside"):
        em.embedding(tokens, w, 1.0, 5)
