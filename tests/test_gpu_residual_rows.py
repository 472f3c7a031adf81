"""A residual with its norms over more rows than the workgroups of a launch take at
once: each of them goes on to further rows, with the next row's values loaded ahead, the
sums of a row of several waves in alternating halves of LDS, and the vectors' sums kept from
row to row.  The last round of rows is not full.  Against the formulas in float64 with the
bounds of test_gpu_residual, here on the GPU."""
import pytest
import torch

import test_gpu_residual as base
from gmdn_amd.residual import residual_norm

pytestmark = pytest.mark.gpu
B, F = torch.bfloat16, torch.float32


def _close(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol + torch.finfo(got.dtype).eps / 2 * (ref.abs() + tol) + 1e-38)
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err - tol).max()):.3e}"


def _run(rows, d, x_dtype, y_dtype, parts, seed):
    dev = base._dev()
    v, dr, dz = base._data(rows, d, seed, x_dtype, y_dtype, parts)
    leaf = {k: t.to(dev).requires_grad_(True) for k, t in v.items() if t is not None}
    v = {k: leaf[k].detach() if t is not None else None for k, t in v.items()}
    dr, dz = dr.to(dev), dz.to(dev)
    (r, tr), (z, tz), state = base._forward(v, 1e-6)
    got_r, got_z = residual_norm(leaf["x"], leaf["y"], leaf["weight"],
                                 **{k: leaf.get(k) for k in ("post_weight", "gate", "scale")})
    _close(got_r.detach(), r, tr, "r")
    _close(got_z.detach(), z, tz, "z")
    grads = dict(zip(leaf, torch.autograd.grad([got_r, got_z], list(leaf.values()), [dr, dz])))
    ref = base._backward(v, dr, dz, state)
    for name, g in grads.items():
        _close(g, *ref[name], "d" + name)


# rows of 64, 128, 256 and 512 threads, two pieces each, in workgroups of 8, 4, 2 and 1 row
@pytest.mark.parametrize("x_dtype,y_dtype", base.PAIRS)
@pytest.mark.parametrize("rows,d", [(4131, 1024), (2100, 2000), (1030, 4000), (1030, 8192), (515, 5001)])
def test_sum(rows, d, x_dtype, y_dtype):
    _run(rows, d, x_dtype, y_dtype, "add", rows + d)


# rows of 128 to 1024 threads, one piece each, in workgroups of 4, 2, 1 and 1 row
@pytest.mark.parametrize("parts", ["post", "scale", "gate", "full"])
@pytest.mark.parametrize("x_dtype,y_dtype", base.PAIRS)
@pytest.mark.parametrize("rows,d", [(2100, 1024), (1100, 2000), (530, 4000), (600, 8192), (515, 5001)])
def test_parts(rows, d, x_dtype, y_dtype, parts):
    _run(rows, d, x_dtype, y_dtype, parts, rows + d)
