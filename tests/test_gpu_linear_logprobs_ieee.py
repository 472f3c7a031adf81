"""Log probabilities from float32 hidden states in 'ieee': the products leave float32's
rounding.

Three pieces of an operand leave 2^-24 of it (each rounding off at most 2^-8 of what is left;
in fact 2^-9); the three products of small pieces that are left out are another two 2^-24,
and so are the two operands: five 2^-24 A in all, and a term is six sums.  A product of one
term only is then within 16 2^-24.  Of random operands the roundings of a sum of K
terms in six products add up to about sqrt(K) 2^-24 of its norm, 5e-7
for the 64 here; the gradient of the logits brings a few 2^-24 of its own.  Together
they stay below 2^-19, where the pieces of 'tf32' (2^-18 each, and the product left out) are
not: about 4e-6."""
import pytest
import torch

import test_gpu_linear_logprobs_tiles as base
from gmdn_amd import logprobs as lpm
from gmdn_amd import scan

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SPLIT = (U, 5 * U, 6)


@pytest.fixture
def ieee():
    before = scan.get_precision()
    scan.set_precision("ieee")
    yield
    scan.set_precision(before)


@pytest.mark.parametrize("rows,V,D", [(1, 1, 1), (3, 5, 7), (70, 70, 70), (130, 257, 256), (200, 33, 100), (1500, 3001, 200),
                                      (1021, 32003, 1001), (2049, 65812, 200)])
def test_forward_backward(rows, V, D):
    base.run(rows, V, D, torch.float32, rows + V + D, split=SPLIT, precision="ieee")


def test_peaked_distributions():
    base.run(40, 300, 64, torch.float32, 8, split=SPLIT, spread=80.0, precision="ieee")


def _norms(**kw):
    x, w, tokens, dl, dh = base.data(64, 64, 64, torch.float32, 1)
    leaf = [t.requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(lpm.linear_logprobs(*leaf, tokens, **kw), leaf, [dl, dh])
    x64, w64 = (t.detach().double().requires_grad_(True) for t in (x, w))
    logp = torch.log_softmax(x64 @ w64.t(), 1)
    kept = tokens != base.IGNORE
    lp = torch.where(kept, logp.gather(1, tokens.clamp(0)[:, None])[:, 0], 0.0)
    want = torch.autograd.grad([lp, torch.special.entr(logp.exp()).sum(1)], [x64, w64], [dl.double(), dh.double()])
    return [float((a.double() - b).norm() / b.norm()) for a, b in zip(got, want)], got


def test_the_setting_is_read(ieee):
    """By the forward; its backward goes on in what the forward had."""
    by_setting, got = _norms()
    assert max(by_setting) < 2.0 ** -19
    assert all(torch.equal(a, b) for a, b in zip(got, _norms(precision="ieee")[1]))
    assert min(_norms(precision="tf32")[0]) > 2.0 ** -19
    x, w, tokens, dl, dh = base.data(64, 64, 64, torch.float32, 1)
    leaf = [t.requires_grad_(True) for t in (x, w)]
    out = lpm.linear_logprobs(*leaf, tokens)
    scan.set_precision("tf32")
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(out, leaf, [dl, dh])))
    assert min(_norms()[0]) > 2.0 ** -19


def test_one_term():
    """Rows of x with one value: a logit is one product, and the largest is kept as it is."""
    dev = base.dev()
    gen = torch.Generator().manual_seed(3)
    x, w = torch.zeros(200, 70), torch.randn(300, 70, generator=gen)
    x[torch.arange(200), torch.arange(200) % 70] = torch.randn(200, generator=gen)
    _, _, stats = torch.ops.gmdn.linear_logprobs_fwd(x.to(dev), w.to(dev), torch.zeros(200, dtype=torch.int64, device=dev),
                                                     -100, 1)
    top = (x.double() @ w.double().t()).amax(1)
    assert ((stats[:, 0].double().cpu() - top).abs() <= 16 * U * top.abs()).all()


def test_bfloat16_operands_do_not_change(ieee):
    x, w, tokens, dl, dh = base.data(70, 200, 64, torch.bfloat16, 2)
    leaf = [t.requires_grad_(True) for t in (x, w)]

    def call(**kw):
        out = lpm.linear_logprobs(*leaf, tokens, **kw)
        return *out, *torch.autograd.grad(out, leaf, [dl, dh])

    assert all(torch.equal(a, b) for a, b in zip(call(), call(precision="tf32")))


def test_refusals():
    x, w, tokens, _, _ = base.data(3, 5, 8, torch.float32, 4)
    with pytest.raises(ValueError, match="'tf32' or 'ieee'"):
        lpm.linear_logprobs(x, w, tokens, precision="fp16")
    with pytest.raises(RuntimeError, match="precision is 0"):
        torch.ops.gmdn.linear_logprobs_fwd(x, w, tokens, -100, 2)
