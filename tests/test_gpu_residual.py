"""GPU parity of a branch's residual with its norms (csrc/residual_norm.hip),
forward and backward, against the formulas in float64.

Bounds, with u = 2^-24.  A sum over a row passes through at most 16 additions in a
thread and ten joining ones: 32 u of its sum of magnitudes; the inverse root, the
logistic function (its argument within 2 u |g|, |g| below 8 here) and the products
that follow stay within ROW = 64 u of each value.  z and the gradients see the
unrounded r's error through the norm.  A vector's gradient adds up to rows / 1024 + 64
products in sequence.  An output adds half a step of its type."""
import pytest
import torch

from gmdn_amd import ops  # noqa: F401
from gmdn_amd.residual import residual_norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROW = 64 * U
B, F = torch.bfloat16, torch.float32
PAIRS = [(B, B), (F, F), (F, B)]
PARTS = ["add", "post", "scale", "gate", "full"]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _close(got, ref, tol, what):
    err = (got.double().cpu() - ref).abs()
    half = torch.finfo(got.dtype).eps / 2
    bad = ~(err <= tol + half * (ref.abs() + tol) + 1e-38)
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err - tol).max()):.3e}"


def _data(rows, d, seed, x_dtype, y_dtype, parts, w_dtype=F, weight=True):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen)

    full = parts == "full"
    v = {"x": (2 * rand(rows, d)).to(x_dtype), "y": rand(rows, d).to(y_dtype),
         "weight": (1 + 0.2 * rand(d)).to(w_dtype) if weight else None,
         "post_weight": (1 + 0.2 * rand(d)).to(w_dtype) if full or parts == "post" else None,
         "gate": rand(rows, d).to(y_dtype) if full or parts == "gate" else None,
         "scale": (0.5 + 0.2 * rand(d)).to(w_dtype) if full or parts == "scale" else None}
    return v, rand(rows, d).to(x_dtype), rand(rows, d).to(y_dtype)


def _forward(v, eps):
    """(value, bound) of r and z, and what the backward takes from them."""
    x, y = v["x"].double(), v["y"].double()
    rho, yh = None, y
    if v["post_weight"] is not None:
        rho = torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
        yh = y * rho
    n = yh if v["post_weight"] is None else yh * v["post_weight"].double()
    u = torch.sigmoid(v["gate"].double()) if v["gate"] is not None else torch.ones_like(y)
    s = v["scale"].double() if v["scale"] is not None else torch.ones_like(y)
    r = x + s * u * n
    tol = ROW * (s * u * n).abs() + 2 * U * r.abs()
    tau = torch.rsqrt((r * r).mean(-1, keepdim=True) + eps)
    w = v["weight"].double() if v["weight"] is not None else torch.ones_like(y)
    z = r * tau * w
    tol_z = (w * tau).abs() * tol + z.abs() * (ROW + tau * tol.amax(-1, keepdim=True))
    th = tau * tol + z.abs() / w.abs() * (ROW + tau * tol.amax(-1, keepdim=True))  # of r tau
    return (r, tol), (z, tol_z), (yh, rho, n, u, s, w, tau, r * tau, th)


def _backward(v, dr, dz, state):
    yh, rho, n, u, s, w, tau, rh, th = state
    dr, dz = dr.double(), dz.double()
    g = w * dz
    G, H = g.abs().amax(-1, keepdim=True), th.amax(-1, keepdim=True)
    dx = dr + tau * (g - rh * (g * rh).mean(-1, keepdim=True))
    tx = 2 * U * dr.abs() + tau * G * (8 * ROW * (1 + rh.abs() + rh * rh) + 3 * H * (1 + rh.abs()))
    dn = dx * s * u
    tn = tx * (s * u).abs() + ROW * dn.abs()
    out = {"x": (dx, tx), "y": (dn, tn)}
    seq = (dx.shape[0] / 1024 + 64) * U
    out["weight"] = ((dz * rh).sum(0), (dz.abs() * (th + (seq + 2 * ROW) * rh.abs())).sum(0))
    if rho is not None:
        p = v["post_weight"].double()
        q, tq = p * dn, p.abs() * tn + U * (p * dn).abs()
        mean = (q * yh).mean(-1, keepdim=True)
        tm = (tq * yh.abs() + 2 * ROW * (q * yh).abs()).mean(-1, keepdim=True)
        dy = rho * (q - yh * mean)
        out["y"] = (dy, rho * (tq + yh.abs() * tm) + 4 * ROW * rho * (q.abs() + (yh * mean).abs()))
        out["post_weight"] = ((dn * yh).sum(0), (tn * yh.abs() + (seq + 2 * ROW) * (dn * yh).abs()).sum(0))
    if v["scale"] is not None:
        out["scale"] = ((dx * u * n).sum(0), (tx * (u * n).abs() + (seq + 2 * ROW) * (dx * u * n).abs()).sum(0))
    if v["gate"] is not None:
        k = s * n * u * (1 - u)
        # 1 - u loses what u's rounding is of it: within ROW of u itself
        out["gate"] = (dx * k, tx * k.abs() + 4 * ROW * (dx * k).abs() + ROW * (dx * s * n * u).abs())
    return out


def _run(rows, d, x_dtype, y_dtype, parts, seed, w_dtype=F, weight=True, use=(True, True), eps=1e-6, pad=0):
    dev = _dev()
    v, dr, dz = _data(rows, d, seed, x_dtype, y_dtype, parts, w_dtype, weight)
    (r, tr), (z, tz), state = _forward(v, eps)

    def place(t):  # as a slice of a wider matrix
        if not pad or t.dim() < 2:
            return t.to(dev)
        return torch.cat([t, torch.full((rows, pad), float("nan"), dtype=t.dtype)], 1).to(dev)[:, :d]

    leaf = {k: place(t).requires_grad_(True) for k, t in v.items() if t is not None}
    named = {k: leaf.get(k) for k in ("post_weight", "gate", "scale")}
    got_r, got_z = residual_norm(leaf["x"], leaf["y"], leaf.get("weight"), eps=eps, **named)
    assert got_r.dtype == x_dtype and got_z.dtype == y_dtype
    _close(got_r.detach(), r, tr, "r")
    _close(got_z.detach(), z, tz, "z")
    outs = [t for t, on in zip((got_r, got_z), use) if on]
    cots = [place(t) for t, on in zip((dr, dz), use) if on]
    grads = dict(zip(leaf, torch.autograd.grad(outs, list(leaf.values()), cots, allow_unused=True)))
    dr, dz = (t if on else torch.zeros_like(t) for t, on in zip((dr, dz), use))
    ref = _backward(v, dr, dz, state)
    for name, g in grads.items():
        assert g.dtype == leaf[name].dtype and g.shape == leaf[name].shape
        _close(g, *ref[name], "d" + name)


SIZES = [(1, 1), (3, 5), (8, 64), (7, 65), (300, 96), (5, 200), (3, 513), (33, 1000), (5, 1001), (1100, 256), (9, 1500),
         (130, 2048), (5, 3000), (9, 4097), (6, 8192)]


@pytest.mark.parametrize("x_dtype,y_dtype", PAIRS)
@pytest.mark.parametrize("rows,d", SIZES)
def test_all_parts(rows, d, x_dtype, y_dtype):
    for parts in PARTS:
        _run(rows, d, x_dtype, y_dtype, parts, rows + d)


@pytest.mark.parametrize("parts", PARTS)
def test_one_output_used(parts):
    for use in ((True, False), (False, True)):
        _run(40, 200, F, F, parts, 1, use=use)
        _run(5, 1001, F, B, parts, 2, use=use)


@pytest.mark.parametrize("parts", PARTS)
def test_bfloat16_vectors_and_none(parts):
    _run(70, 300, B, B, parts, 3, w_dtype=B)
    _run(70, 300, F, B, parts, 4, weight=False)


@pytest.mark.parametrize("parts", PARTS)
def test_slices_of_wider_matrices(parts):
    _run(37, 129, B, B, parts, 5, pad=3)
    _run(6, 1024, F, F, parts, 6, pad=8)
    _run(3, 5001, F, B, parts, 7, pad=1)


def test_many_rows():
    _run(20000, 40, F, B, "full", 8)
    _run(9000, 300, B, B, "add", 9)


def test_differences():
    """The gradients beside differences of the operator itself in float32."""
    dev = _dev()
    v, _, _ = _data(4, 12, 10, F, F, "full")
    leaf = {k: t.to(dev).requires_grad_(True) for k, t in v.items()}
    gen = torch.Generator().manual_seed(11)
    a, b = (torch.randn(4, 12, generator=gen).to(dev) for _ in range(2))

    def value():
        r, z = residual_norm(leaf["x"], leaf["y"], leaf["weight"], post_weight=leaf["post_weight"], gate=leaf["gate"],
                             scale=leaf["scale"])
        return (r * a).double().sum() + (z * b).double().sum()

    grads = torch.autograd.grad(value(), list(leaf.values()))
    h = 2.0 ** -7  # differences are off by h^2 / 6 of a third derivative, and by 2^-24 / h of values below 100
    for t, g in zip(leaf.values(), grads):
        at = t.detach().view(-1)
        for i in range(0, at.numel(), 5):
            keep = at[i].item()
            with torch.no_grad():
                at[i] = keep + h
                up = value()
                at[i] = keep - h
                down = value()
                at[i] = keep
            assert abs(float(up - down) / (2 * h) - float(g.view(-1)[i])) < 5e-3


def test_rows_of_zeros_and_large_values():
    """A row of zeros norms to zeros; one near the type's end stays finite where
    its square does; NaN and infinities stay in their rows."""
    dev = _dev()
    x, y = torch.zeros(6, 96), torch.zeros(6, 96)
    x[1], x[2, 3], x[3, 5], y[4, 7] = 1e15, float("nan"), float("inf"), float("nan")
    x[5], y[5] = 1.0, 2.0
    one = torch.ones(96)
    xd, yd = x.to(dev).requires_grad_(True), y.to(dev).requires_grad_(True)
    r, z = residual_norm(xd, yd, one.to(dev), post_weight=one.to(dev), eps=1e-6)
    assert (z[0] == 0).all() and torch.allclose(z[1], torch.ones_like(z[1])) and z[2].isnan().all() and z[4].isnan().all()
    assert torch.allclose(z[5], torch.ones_like(z[5]))
    dx, dy = torch.autograd.grad([r, z], [xd, yd], [torch.ones_like(r), torch.ones_like(z)])
    for i in (0, 1, 5):
        assert dx[i].isfinite().all() and dy[i].isfinite().all()


def test_no_rows():
    dev = _dev()
    v, _, _ = _data(0, 24, 0, F, B, "full")
    leaf = {k: t.to(dev).requires_grad_(True) for k, t in v.items()}
    r, z = residual_norm(leaf["x"], leaf["y"], leaf["weight"], post_weight=leaf["post_weight"], gate=leaf["gate"],
                         scale=leaf["scale"])
    grads = torch.autograd.grad([r, z], list(leaf.values()), [torch.empty_like(r), torch.empty_like(z)])
    assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, leaf.values()))


def test_shared_gradient_is_not_written_twice():
    """Without any part the stream's and the branch's gradients are one tensor:
    adding to one's leaf must not change the other's."""
    dev = _dev()
    x, y = (torch.randn(5, 64).to(dev).requires_grad_(True) for _ in range(2))
    r, z = residual_norm(x, y)
    ((r + z).sum() + 3 * x.sum()).backward()
    once = y.grad.clone()
    assert torch.allclose(x.grad, once + 3, rtol=1e-6, atol=1e-6)
    r, z = residual_norm(x, y)
    (r + z).sum().backward()
    assert torch.allclose(y.grad, 2 * once, rtol=1e-6, atol=1e-6)
    assert torch.allclose(x.grad, 2 * once + 3, rtol=1e-6, atol=1e-6)


def test_refusals():
    dev = _dev()
    x, w = torch.randn(3, 8, device=dev), torch.ones(8, device=dev)
    for call, message in [
            (lambda: residual_norm(x.half(), x.half()), "bfloat16 or float32"),
            (lambda: residual_norm(x.bfloat16(), x), "failed with code 2"),
            (lambda: residual_norm(x, x[:2]), "shape"),
            (lambda: residual_norm(x, x, w[:4]), "shape"),
            (lambda: residual_norm(x, x, w, scale=w.bfloat16()), "of one type"),
            (lambda: residual_norm(x, x, w, gate=x.bfloat16()), "gate is"),
            (lambda: residual_norm(x, x, w, gate=x[:, :1]), "shape"),
            (lambda: residual_norm(x, x, w.cpu()), "weight is on"),
            (lambda: residual_norm(x, x, w, eps=-1.0), "failed with code 1"),
            (lambda: residual_norm(x, x, w, eps=float("nan")), "failed with code 1"),
            (lambda: residual_norm(torch.ones(1, 8193, device=dev), torch.ones(1, 8193, device=dev)),
             "failed with code 2")]:
        with pytest.raises(RuntimeError, match=message):
            call()
