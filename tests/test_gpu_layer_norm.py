"""GPU parity of layer norm, forward and backward, and of the same from an
8-bit checkpoint of its input (csrc/layer_norm.hip), against the formulas in
float64.

Bounds.  A sum over a row passes through at most 16 additions in a thread and
ten joining ones, so with u = 2^-24 a sum's relative error (to the sum of
magnitudes) is below 32 u; mean, deviation and normalised value then differ
by a few such terms: ROW = 64 u covers each.  A weight gradient adds up to
rows / 1024 + 64 products in sequence.  An output in bfloat16 adds half a unit
in its last place."""
import pytest
import torch

from gmdn_amd import layer_norm as ln
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROW = 64 * U
PAIRS = [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float32, torch.bfloat16)]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def rounding(ref, dtype):
    """Half a unit in the last place of `dtype` at the reference's values."""
    bits = 8 if dtype == torch.bfloat16 else 24
    return torch.pow(2.0, torch.floor(torch.log2(ref.abs().clamp_min(1e-300))) - bits)


def assert_close(got, ref, tol, what):
    err = (got.double().cpu() - ref).abs()
    bad = ~(err <= tol + rounding(ref, got.dtype) * (1 + 2 ** -6) + 1e-38)
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err - tol).max()):.3e}"


def reference(x, w, b, dy, eps):
    """y, dx, dweight, dbias in float64 by the formulas, with their bounds.
    x may be what the checkpoint reads back as beside the true statistics."""
    x, true = x if isinstance(x, tuple) else (x, x)
    mean = true.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((true - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * r
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b
    g = dy * w
    mg, mx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    tol_xh = ROW * (r * true.abs().amax(-1, keepdim=True) + 3 * xh.abs())
    tx = tol_xh.amax(-1, keepdim=True)
    G = g.abs().amax(-1, keepdim=True)
    seq = (x.shape[0] / 1024 + 64) * U
    return {
        "y": (xh * w + b, tol_xh * w.abs() + 4 * U * (xh * w).abs() + 4 * U * b.abs()),
        "dx": (r * (g - mg - xh * mx), r * G * (4 * ROW * (1 + xh.abs()) + tx * (1 + 2 * xh.abs()))),
        "dw": ((dy * xh).sum(0), (dy.abs() * (tol_xh + seq * xh.abs())).sum(0)),
        "db": (dy.sum(0), seq * dy.abs().sum(0)),
        "mean": (mean[:, 0], ROW * true.abs().mean(-1)),
        "rstd": (r[:, 0], ROW * r[:, 0] * (1 + r[:, 0] * true.abs().amax(-1))),
    }


def data(rows, d, seed, x_dtype, y_dtype, w_dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d, generator=gen) * (1 + 9 * (torch.rand(d, generator=gen) < 0.02)) + 0.3
    w, b = 1 + 0.2 * torch.randn(d, generator=gen), 0.2 * torch.randn(d, generator=gen)
    dy = torch.randn(rows, d, generator=gen)
    return x.to(x_dtype), w.to(w_dtype), b.to(w_dtype), dy.to(y_dtype)


SIZES = [(1, 1), (3, 5), (8, 64), (7, 65), (300, 96), (1, 1024), (33, 1000), (5, 1001), (1100, 256), (130, 2048),
         (9, 4097), (6, 8192), (3, 16384), (5, 16383)]


@pytest.mark.parametrize("x_dtype,y_dtype", PAIRS)
@pytest.mark.parametrize("rows,d", SIZES)
def test_forward_backward(rows, d, x_dtype, y_dtype):
    dev = _dev()
    x, w, b, dy = data(rows, d, rows + d, x_dtype, y_dtype)
    ref = reference(x.double(), w.double(), b.double(), dy.double(), 1e-5)
    xd, wd, bd = (t.to(dev).requires_grad_(True) for t in (x, w, b))
    y = ln.layer_norm(xd, wd, bd, dtype=y_dtype)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(dev))
    assert y.dtype == y_dtype and dx.dtype == x_dtype and dw.dtype == db.dtype == torch.float32
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert_close(got, *ref[name], name)
    _, mean, rstd, q, scale = torch.ops.gmdn.layer_norm_fwd(xd, wd, bd, 1e-5, y_dtype, False)
    assert q.numel() == scale.numel() == 0
    assert_close(mean, *ref["mean"], "mean")
    assert_close(rstd, *ref["rstd"], "rstd")


@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", ["none", "weight", "both"])
def test_optional_and_bfloat16_weights(which, w_dtype):
    dev = _dev()
    x, w, b, dy = data(40, 200, 3, torch.bfloat16, torch.bfloat16, w_dtype)
    w, b = w if which != "none" else None, b if which == "both" else None
    ref = reference(x.double(), None if w is None else w.double(), None if b is None else b.double(), dy.double(), 1e-5)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b) if t is not None]
    y = ln.layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy.to(dev))
    assert_close(y, *ref["y"], "y")
    for name, got in zip(("dx", "dw", "db"), grads):
        assert_close(got, *ref[name], name)
    assert all(g.dtype == w_dtype for g in grads[1:])


@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", [(1, 200), (16, 200), (128, 200), (129, 200), (32, 1000), (33, 1000), (16, 1500),
                                    (4, 5001), (5, 5001), (4, 16384)])
def test_weight_gradients_of_few_rows(rows, d, w_dtype):
    """One workgroup writes them itself up to a number of rows; past it their
    sums go through memory."""
    dev = _dev()
    x, w, b, dy = data(rows, d, rows + d, torch.float32, torch.bfloat16, w_dtype)
    ref = reference(x.double(), w.double(), b.double(), dy.double(), 1e-5)
    args = [t.to(dev) for t in (x, w, b)]
    _, mean, rstd, _, _ = torch.ops.gmdn.layer_norm_fwd(*args, 1e-5, torch.bfloat16, False)
    grads = torch.ops.gmdn.layer_norm_bwd(dy.to(dev), args[0], args[1], mean, rstd)
    for name, got in zip(("dx", "dw", "db"), grads):
        assert_close(got, *ref[name], name)
    assert grads[1].dtype == grads[2].dtype == w_dtype


def test_strided_rows_and_gradients():
    """A slice of a wider tensor at an odd offset, a transposed batch and a
    broadcast cotangent give what their contiguous copies give."""
    dev = _dev()
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(6, 7, 211, generator=gen).to(dev)
    w, b = torch.randn(200, generator=gen).to(dev), torch.randn(200, generator=gen).to(dev)
    for x in (wide[..., 3:203], wide.transpose(0, 1)[..., 5:205], wide[::2, :, 11:], wide[0, 0, 1:201]):
        dy = torch.randn(x.shape[-1], generator=gen).to(dev).expand(x.shape)
        got = _grads(x, w, b, dy)
        want = _grads(x.contiguous(), w, b, dy.contiguous())
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        assert got[0].is_contiguous() and got[0].shape == x.shape


def _grads(x, w, b, dy, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = ln.layer_norm(*leaves, **kw)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


def test_constant_and_nonfinite_rows():
    """A row of one value has deviation 0: the output is the bias, finite
    gradients.  A NaN or an infinity makes its own row NaN and no other."""
    dev = _dev()
    x, w, b, dy = (t.to(dev) for t in data(6, 300, 5, torch.float32, torch.float32))
    x[1] = 2.5
    x[3, 7] = float("nan")
    x[4, 299] = float("inf")
    y, dx, dw, db = _grads(x, w, b, dy)
    assert torch.equal(y[1], b) and torch.isfinite(dx[1]).all()
    for t in (y, dx):
        assert t[3].isnan().all() and t[4].isnan().all()
        assert torch.isfinite(t[[0, 1, 2, 5]]).all()
    assert dw.isnan().all() and torch.isfinite(db).all()


def test_no_rows():
    dev = _dev()
    x, w, b = torch.empty(2, 0, 24, device=dev), torch.ones(24, device=dev), torch.zeros(24, device=dev)
    y, dx, dw, db = _grads(x, w, b, torch.empty_like(x))
    assert y.shape == dx.shape == x.shape
    assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


def test_large_mean():
    """Values far from zero: the deviation comes from centred values (a
    difference of squares would lose them all)."""
    dev = _dev()
    x, w, b, dy = data(16, 512, 6, torch.float32, torch.float32)
    x = x + 3000.0
    ref = reference(x.double(), w.double(), b.double(), dy.double(), 1e-5)
    y, dx, dw, db = _grads(*(t.to(dev) for t in (x, w, b, dy)))
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert_close(got, *ref[name], name)


def test_gradient_against_differences():
    """The directional derivative of sum(c y) by central differences of the
    operator's own forward at two steps: their difference bounds the
    truncation, 8 u |c| |y| per value the rounding."""
    dev = _dev()
    gen = torch.Generator().manual_seed(9)
    x, w, b, c = (torch.randn(*s, generator=gen).to(dev) for s in ((4, 50), (50,), (50,), (4, 50)))
    _, *grads = _grads(x, w, b, c)
    for i, g in enumerate(grads):
        v = torch.randn(g.shape, generator=gen).to(dev)

        def loss(h):
            at = [x, w, b]
            at[i] = at[i] + h * v
            y = ln.layer_norm(*at).double()
            return (c.double() * y).sum().item(), (c.double() * y).abs().sum().item()

        def slope(h):
            (p, a), (m, _) = loss(h), loss(-h)
            return (p - m) / (2 * h), 8 * U * a / h

        (d1, r1), (d2, r2) = slope(0.02), slope(0.04)
        got = (g.double() * v.double()).sum().item()
        assert abs(got - d1) <= abs(d2 - d1) + r1 + r2 + 1e-5 * abs(got), (i, got, d1, d2)


def kept(x):
    """What the checkpoint of x reads back as, by the format's definition, in float64."""
    out = torch.empty(x.shape, dtype=torch.float64)
    x = x.float()
    for a in range(0, x.shape[-1], 128):
        v = x[..., a:a + 128]
        amax = v.abs().amax(-1, keepdim=True)
        q = torch.round(v * (torch.full_like(amax, 127.0) / amax))
        out[..., a:a + 128] = torch.where(amax < 2.0 ** -100, 0.0,
                                          q.double() * (amax * float.fromhex("0x1.020406p-7")).double())
    return out


@pytest.mark.parametrize("x_dtype,y_dtype", PAIRS)
@pytest.mark.parametrize("rows,d", [(3, 5), (9, 64), (7, 200), (33, 1000), (5, 1001), (40, 1024), (4, 5000), (3, 16384)])
def test_from_checkpoint(rows, d, x_dtype, y_dtype):
    """The backward from the 8-bit checkpoint: the formulas at what it reads
    back as, with the true input's statistics; the rebuilt output likewise.
    (Reading back: one product, relative error u.)"""
    dev = _dev()
    x, w, b, dy = data(rows, d, rows * d, x_dtype, y_dtype)
    back = kept(x)
    ref = reference((back, x.double()), w.double(), b.double(), dy.double(), 1e-5)
    xd, wd, bd = (t.to(dev).requires_grad_(True) for t in (x, w, b))
    y = ln.layer_norm(xd, wd, bd, dtype=y_dtype, checkpoint="int8")
    assert torch.equal(y, ln.layer_norm(xd, wd, bd, dtype=y_dtype))
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(dev))
    assert dx.dtype == x_dtype
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        assert_close(got, *ref[name], name)
    with torch.no_grad():
        _, mean, rstd, q, scale = torch.ops.gmdn.layer_norm_fwd(xd, wd, bd, 1e-5, y_dtype, True)
        want_q, want_scale = torch.ops.gmdn.act8_pack(xd)
        assert torch.equal(q, want_q) and torch.equal(scale, want_scale)
        again = torch.ops.gmdn.layer_norm8_rebuild(q, scale, wd, bd, mean, rstd, y_dtype)
    assert_close(again, *ref["y"], "rebuilt")


@pytest.mark.parametrize("dtype,rows,d", [(torch.bfloat16, 13000, 4000), (torch.float32, 13000, 2048),
                                          (torch.float32, 3000, 1024)])
def test_large_matrices_equal_their_parts(dtype, rows, d):
    """From 96 MB on a matrix goes past the caches, below it a float32 dx does:
    the same bits as its parts, which are on the other side or the same."""
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(rows, d, generator=gen, device=dev).to(dtype)
    dy = torch.randn(rows, d, generator=gen, device=dev).to(dtype)
    w, b = torch.randn(d, generator=gen, device=dev), torch.randn(d, generator=gen, device=dev)

    def rows_of(x, dy):
        y, mean, rstd, q, scale = torch.ops.gmdn.layer_norm_fwd(x, w, b, 1e-5, dtype, True)
        return (y, mean, rstd, q, scale, torch.ops.gmdn.layer_norm_bwd(dy, x, w, mean, rstd)[0],
                torch.ops.gmdn.layer_norm8_bwd(dy, q, scale, w, mean, rstd, dtype)[0],
                torch.ops.gmdn.layer_norm8_rebuild(q, scale, w, b, mean, rstd, dtype))

    whole = rows_of(x, dy)
    for a in (0, rows - 500):
        part = rows_of(x[a:a + 500], dy[a:a + 500])
        assert all(torch.equal(o[a:a + 500], p) for o, p in zip(whole, part))


def test_deterministic_and_on_another_stream():
    dev = _dev()
    x, w, b, dy = (t.to(dev) for t in data(5000, 1024, 2, torch.float32, torch.bfloat16))
    first = _grads(x, w, b, dy, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _grads(x, w, b, dy, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, second))


def test_module_matches_torch_under_autocast():
    """Under bfloat16 autocast the module's output is torch's float32 norm
    rounded to bfloat16."""
    dev = _dev()
    torch.manual_seed(0)
    mine, theirs = ln.LayerNorm(384).to(dev), torch.nn.LayerNorm(384).to(dev)
    x = torch.randn(3, 17, 384, device=dev)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, ref = mine(x), theirs(x)
    assert y.dtype == torch.bfloat16 and ref.dtype == torch.float32
    xh = ref.double().cpu()
    assert_close(y, xh, 2 * ROW * (xh.abs() + 4), "autocast")
    assert mine(x).dtype == torch.float32
    mine.load_state_dict(theirs.state_dict())


def test_refusals():
    dev = _dev()
    x, w, b = torch.randn(4, 16, device=dev), torch.ones(16, device=dev), torch.zeros(16, device=dev)
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        ln.layer_norm(x.half(), w, b)
    with pytest.raises(RuntimeError, match="unsupported"):
        ln.layer_norm(x.bfloat16(), w, b, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="weight has shape"):
        ln.layer_norm(x, w[:8], b[:8])
    with pytest.raises(RuntimeError, match="bias is"):
        ln.layer_norm(x, w, b.bfloat16())
    with pytest.raises(RuntimeError, match="comes with a weight"):
        ln.layer_norm(x, None, b)
    with pytest.raises(RuntimeError, match="weight is on"):
        ln.layer_norm(x, w.cpu(), b.cpu())
    with pytest.raises(RuntimeError, match="invalid argument"):
        ln.layer_norm(x, w, b, eps=-1.0)
    with pytest.raises(RuntimeError, match="at least one value"):
        ln.layer_norm(x[:, :0], None)
    with pytest.raises(RuntimeError, match="unsupported"):
        ln.layer_norm(torch.zeros(1, 16385, device=dev))
    with pytest.raises(ValueError, match="int8"):
        ln.layer_norm(x, checkpoint="int4")
    y, mean, rstd, _, _ = torch.ops.gmdn.layer_norm_fwd(x, w, b, 1e-5, torch.float32, False)
    with pytest.raises(RuntimeError, match="mean has shape"):
        torch.ops.gmdn.layer_norm_bwd(y, x, w, mean[:3], rstd)
    with pytest.raises(RuntimeError, match="x has shape"):
        torch.ops.gmdn.layer_norm_bwd(y, x[:3], w, mean, rstd)
    x.requires_grad_(True)
    dx = torch.autograd.grad(ln.layer_norm(x, w, b).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="layer_norm_bwd"):
        dx.sum().backward()
