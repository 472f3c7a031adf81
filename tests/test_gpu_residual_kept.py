"""Gradients of a residual whose results the caller goes on changing."""
import pytest
import torch

from gmdn_amd import ops  # noqa: F401
from gmdn_amd.residual import residual_norm

pytestmark = pytest.mark.gpu
B, F = torch.bfloat16, torch.float32


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


@pytest.mark.parametrize("y_dtype", [F, B])
def test_norm_changed_in_place(y_dtype):
    """The gradients are those of the same product out of place, bit for bit."""
    dev = _dev()
    gen = torch.Generator().manual_seed(1)
    x, y, w = (torch.randn(*n, generator=gen).to(t).to(dev).requires_grad_(True)
               for n, t in (((70, 200), F), ((70, 200), y_dtype), ((200,), F)))
    dr, dz = torch.randn(70, 200, generator=gen).to(dev), torch.randn(70, 200, generator=gen).to(y_dtype).to(dev)

    def grads(change):
        r, z = residual_norm(x, y, w)
        return torch.autograd.grad([r, change(z)], [x, y, w], [dr, dz])

    for a, b in zip(grads(lambda z: z.mul_(2)), grads(lambda z: z * 2)):
        assert torch.equal(a, b)


def test_a_branch_is_asked_for_where_it_is_read():
    dev = _dev()
    x, w, s = torch.randn(6, 64, device=dev), torch.ones(64, device=dev), torch.ones(6, device=dev)
    op = torch.ops.gmdn.residual_norm_bwd
    for args in ((x.to(B), None, x.to(B), None, w, None, None, None, s, s[:0]),
                 (x, None, x, None, w, None, None, w, s, s[:0]),
                 (x, None, x, None, w, None, x, None, s, s[:0])):
        with pytest.raises(RuntimeError, match="y is given"):
            op(*args)
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        op(x, None, x, None, w, None, None, None, s, s[:0], torch.float16)
