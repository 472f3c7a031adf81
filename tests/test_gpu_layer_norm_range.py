"""Layer norm's backward of rows near the ends of float32's range, against the
formulas in float64."""
import pytest
import torch

from gmdn_amd import layer_norm as ln
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("d", [1, 70, 200, 600, 1500, 5001])
def test_rows_of_one_large_value(d, sign):
    """x = 2^112 throughout: the mean is exact (every partial sum is an integer
    of at most 13 bits times 2^112), the deviation 0, and with eps = 1e-35
    1 / deviation is 3.2e17, their product past the largest float32.  So y = b
    and dx = (g - mean(g)) / sqrt(eps), in sums of at most 32 terms in
    sequence, and finite: a column past the row's end must not count."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    gen = torch.Generator().manual_seed(d)
    w, b, dy = 1 + 0.2 * torch.randn(d, generator=gen), torch.randn(d, generator=gen), torch.randn(300, d, generator=gen)
    x = torch.full((300, d), sign * 2.0 ** 112)
    x[1:] = torch.randn(299, d, generator=gen)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = ln.layer_norm(*leaves, eps=1e-35)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.cuda())
    assert torch.equal(y[0].cpu(), b)
    g = dy[0].double() * w.double()
    want = (g - g.mean()) / torch.tensor(1e-35, dtype=torch.float32).double().sqrt()
    bound = 64 * U * g.abs().max() / 1e-35 ** 0.5
    assert ((dx[0].double().cpu() - want).abs() <= bound).all()
    assert all(torch.isfinite(t).all() for t in (dx, dw, db))
