"""GPU parity of layer norm's weight gradients where many workgroups' partial
sums are added (csrc/layer_norm.hip, ln_bwd and ln_sums): more than 128 of
them, and a full grid whose threads take several rows, the last turn uneven.
Against the formulas in float64, under the bounds of the other sizes: a thread
adds its rows (3 at most here), a workgroup up to 64 of them side by side,
then two partial sums in turn and twenty joins: below the 64 products in
sequence that they allow."""
import pytest
import torch

from gmdn_amd import layer_norm as ln
from gmdn_amd import ops  # noqa: F401
from test_gpu_layer_norm import assert_close, data, kept, reference

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
# (rows, d): 138 workgroups; 256 of 8 rows, three turns, the last of 3 rows;
# 256 of one row, three turns; two turns; 256 of 64 rows, two turns
SIZES = [(1100, 1024), (4099, 1001), (700, 5001), (300, 16384), (17000, 60)]


@pytest.mark.parametrize("source", ["x", "int8"])
@pytest.mark.parametrize("x_dtype,y_dtype,w_dtype", [(F32, BF16, F32), (BF16, BF16, BF16), (F32, F32, F32)])
@pytest.mark.parametrize("rows,d", SIZES)
def test_gradients_of_many_rows(rows, d, x_dtype, y_dtype, w_dtype, source):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    x, w, b, dy = data(rows, d, rows + d, x_dtype, y_dtype, w_dtype)
    at = (kept(x), x.double()) if source == "int8" else x.double()
    ref = reference(at, w.double(), b.double(), dy.double(), 1e-5)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = ln.layer_norm(*leaves, dtype=y_dtype, checkpoint=None if source == "x" else "int8")
    for name, got in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy.cuda())):
        assert_close(got, *ref[name], name)
