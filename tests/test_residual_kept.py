"""What a residual with its norms keeps for its backward (meta tensors: no kernel
runs).  A float32 stream with nothing but the sum keeps the stream that it returns,
the norm's weight and the rows' statistics: neither the branch's output nor the norm's
result, which the caller may change or free."""
import pytest
import torch

from gmdn_amd import ops  # noqa: F401
from gmdn_amd.residual import residual_norm

B, F = torch.bfloat16, torch.float32


def _kept(call):
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        out = call()
    return out, kept


def _t(*shape, dtype=F):
    return torch.empty(*shape, dtype=dtype, device="meta").requires_grad_(True)


@pytest.mark.parametrize("y_dtype", [F, B])
def test_a_float32_sum_keeps_one_matrix(y_dtype):
    x, y, w = _t(6, 64), _t(6, 64, dtype=y_dtype), _t(64)
    (r, z), kept = _kept(lambda: residual_norm(x, y, w))
    assert r.dtype == F and z.dtype == y_dtype
    assert [t.dtype for t in kept if t.shape == x.shape] == [F]
    assert sum(t.numel() * t.element_size() for t in kept) == 4 * (6 * 64 + 64 + 6)


@pytest.mark.parametrize("y_dtype", [F, B])
def test_the_norm_may_be_changed_in_place(y_dtype):
    x, y, w = _t(6, 64), _t(6, 64, dtype=y_dtype), _t(64)
    r, z = residual_norm(x, y, w)
    grads = torch.autograd.grad([r, z.mul_(2)], [x, y, w], [torch.empty_like(r), torch.empty_like(z)])
    assert [(g.shape, g.dtype) for g in grads] == [(t.shape, t.dtype) for t in (x, y, w)]


def test_what_is_read_may_not_be_changed():
    x, y, w = _t(6, 64), _t(6, 64), _t(64)
    r, z = residual_norm(x, y, w)
    r.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z, [x, y, w], torch.empty_like(z))


@pytest.mark.parametrize("dtype", [F, B])
def test_with_parts_the_inputs_are_kept(dtype):
    x, y, v = _t(6, 64, dtype=dtype), _t(6, 64, dtype=dtype), _t(64)
    (r, z), kept = _kept(lambda: residual_norm(x, y, v, post_weight=v, scale=v))
    whole = [t for t in kept if t.shape == x.shape]
    assert len(whole) == 2 and not any(t is o for t in whole for o in (r, z))


def test_the_backward_without_a_branch():
    """``y`` may be left out where it is not read, with its type where that is not the
    stream's; elsewhere it is asked for."""
    op = torch.ops.gmdn.residual_norm_bwd
    x, w, s = (torch.empty(*n, device="meta") for n in ((6, 64), (64,), (6,)))
    dx, dy, dw, *rest = op(x, None, x, None, w, None, None, None, s, s[:0])
    assert dx.shape == x.shape and dy.numel() == 0 and dw.shape == w.shape
    dx, dy, *rest = op(x, None, x, None, w, None, None, None, s, s[:0], B)
    assert dy.shape == x.shape and dy.dtype == B
