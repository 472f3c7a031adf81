"""Gradients of the entropy and of the alternatives beside tokens outside the
vocabulary: these outputs do not depend on the token, so their gradients are those of
any other token, bit for bit.  Only the log probability of such a token, and what is
differentiated through it, is NaN."""
import pytest
import torch

from gmdn_amd import logprobs as lpm
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _tokens(rows, V, dev):
    inside = torch.arange(rows, device=dev) % V
    outside = inside.clone()
    outside[:4] = torch.tensor([V, -1, -7, 1 << 40])
    return inside, outside


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_logprobs(dtype):
    dev = _dev()
    gen = torch.Generator().manual_seed(1)
    x, w = (torch.randn(n, 64, generator=gen).to(dtype).to(dev).requires_grad_(True) for n in (20, 50))
    dh = torch.randn(20, generator=gen).to(dev)
    inside, outside = _tokens(20, 50, dev)
    want = torch.autograd.grad(lpm.linear_logprobs(x, w, inside).entropy, [x, w], dh)
    got = lpm.linear_logprobs(x, w, outside)
    assert got.logprob[:4].isnan().all() and got.logprob[4:].isfinite().all()
    for a, b in zip(torch.autograd.grad(got.entropy, [x, w], dh), want):
        assert a.isfinite().all() and torch.equal(a, b)
    (dx,) = torch.autograd.grad(lpm.linear_logprobs(x, w, outside).logprob, x, dh)
    assert dx[:4].isnan().all() and dx[4:].isfinite().all()


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs(dtype, top):
    dev = _dev()
    gen = torch.Generator().manual_seed(2)
    logits = torch.randn(20, 300, generator=gen).to(dtype).to(dev).requires_grad_(True)
    dh, dt = torch.randn(20, generator=gen).to(dev), torch.randn(20, top, generator=gen).to(dev)
    inside, outside = _tokens(20, 300, dev)

    def grad(tokens, *names):
        got = lpm.token_logprobs(logits, tokens, top)
        cots = {"logprob": dh, "entropy": dh, "top_logprobs": dt}
        return torch.autograd.grad([getattr(got, n) for n in names], logits, [cots[n] for n in names])[0]

    for names in (["entropy"], ["entropy", "top_logprobs"], ["top_logprobs"])[:3 if top else 1]:
        want, got = grad(inside, *names), grad(outside, *names)
        assert got.isfinite().all() and torch.equal(got, want)
    got = grad(outside, "logprob")
    assert got[:4].isnan().all() and got[4:].isfinite().all()
