"""GPU parity of the 8-bit activation checkpoints (csrc/act8.hip): the stored
bytes against the format's definition bit for bit, GELU and its derivative
against float64, and the layers built on them.

Bounds.  With u = 2^-24: the normal distribution function by float32's erfc or
an approximation as good is within 32 u relative, plus h^2 u from rounding
the exponent -h^2 / 2; the products after it add a few u."""
import math

import pytest
import torch
import torch.nn.functional as F

from gmdn_amd import act8
from gmdn_amd import ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
STEP = float.fromhex("0x1.020406p-7")
TYPES = [torch.bfloat16, torch.float32]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def definition(x):
    """q and scale of a CPU tensor by the format's definition, in float32."""
    d = x.shape[-1]
    groups = -(-d // 128)
    v = F.pad(x.float(), (0, groups * 128 - d)).reshape(*x.shape[:-1], groups, 128)
    amax = v.abs().amax(-1, keepdim=True)
    zero, finite = amax < 2.0 ** -100, torch.isfinite(amax)
    inverse = torch.full_like(amax, 127.0) / amax
    q = torch.where(~zero & finite, torch.round(v * inverse), 0.0)
    scale = torch.where(zero, 0.0, torch.where(finite, amax * STEP, math.nan))
    return q.to(torch.int8).reshape(*x.shape[:-1], groups * 128)[..., :d], scale[..., 0]


def values(shape, seed, dtype):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=gen))
    return x.to(dtype)


def same(a, b):
    return torch.equal(a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (4, 127), (4, 128), (4, 129), (2, 3, 1000), (33, 1024),
                                   (7, 4097), (2000, 384), (1, 100000), (3, 0 + 255)])
def test_pack_and_unpack(shape, dtype):
    dev = _dev()
    x = values(shape, sum(shape), dtype)
    q, scale = act8.pack(x.to(dev))
    want_q, want_scale = definition(x)
    assert torch.equal(q.cpu(), want_q) and torch.equal(scale.cpu(), want_scale)
    for out in TYPES:
        back = act8.unpack((q, scale), out)
        assert back.dtype == out
        d = shape[-1]
        full = want_q.float() * want_scale.repeat_interleave(128, -1)[..., :d]
        assert torch.equal(back.cpu(), full.to(out))
    amax = F.pad(x.float().abs(), (0, -d % 128)).reshape(*shape[:-1], -1, 128).amax(-1).repeat_interleave(128, -1)[..., :d]
    err = (full.double() - x.double()).abs()
    assert (err <= amax.double() / 254 * (1 + 2 ** -14)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_values(dtype):
    """Zeros, magnitudes below and at 2^-100, the type's largest values, and
    groups that hold an infinity or a NaN; each group by itself."""
    dev = _dev()
    big = torch.finfo(dtype).max
    x = torch.zeros(8, 256, dtype=dtype)
    x[1] = 2.0 ** -101
    x[2] = 2.0 ** -100
    x[3] = torch.where(torch.arange(256) % 3 == 0, -big, 0.75 * big).to(dtype)
    x[4, :128] = 1.0
    x[4, 5] = math.inf
    x[5, 128:] = -2.0
    x[5, 255] = math.nan
    x[6] = torch.finfo(dtype).tiny
    x[7, 3] = -0.0
    x[7, 200] = 1e-3
    q, scale = act8.pack(x.to(dev))
    want_q, want_scale = definition(x)
    assert torch.equal(q.cpu(), want_q) and same(scale.cpu(), want_scale)
    back = act8.unpack((q, scale), dtype).cpu()
    assert back[0].eq(0).all() and back[1].eq(0).all() and back[6].eq(0).all()
    assert back[2].ne(0).all() and torch.isfinite(back[3]).all()
    assert (back[3].double() - x[3].double()).abs().max() <= big / 254 * 1.001 + big * 2.0 ** -9 * (dtype != torch.float32)
    assert back[4, :128].isnan().all() and back[4, 128:].eq(0).all()
    assert back[5, :128].eq(0).all() and back[5, 128:].isnan().all()


def test_strides_and_empty():
    dev = _dev()
    wide = values((6, 5, 403), 1, torch.float32).to(dev)
    for x in (wide[..., 1:301], wide.transpose(0, 1)[..., 2:], wide[::2, ::2], wide[0, 0], wide.transpose(1, 2),
              wide[:, :1].expand(6, 4, 403)):
        q, scale = act8.pack(x)
        want_q, want_scale = definition(x.cpu())
        assert torch.equal(q.cpu(), want_q) and torch.equal(scale.cpu(), want_scale)
    q, scale = act8.pack(torch.empty(0, 40, device=dev))
    assert q.shape == (0, 40) and scale.shape == (0, 1)
    assert act8.unpack((q, scale)).shape == (0, 40)
    assert act8.gelu(torch.empty(3, 0, 40, device=dev)).shape == (3, 0, 40)


def gelu64(h):
    cdf = 0.5 * torch.special.erfc(-h / math.sqrt(2))
    pdf = torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)
    rel = U * (32 + h * h)
    return (h * cdf, (h * cdf).abs() * rel), (cdf + h * pdf, (cdf + h.abs() * pdf) * rel)


def assert_close(got, ref, tol, what):
    bits = 8 if got.dtype == torch.bfloat16 else 24
    half = torch.pow(2.0, torch.floor(torch.log2(ref.abs().clamp_min(1e-300))) - bits)
    err = (got.double().cpu() - ref).abs()
    bad = ~(err <= tol + half * (1 + 2 ** -6) + 2.0 ** -126)
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err - tol).max()):.3e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (4, 128), (5, 129), (2, 3, 1000), (33, 1024), (7, 4097), (600, 512)])
def test_gelu(shape, dtype):
    dev = _dev()
    h = (2 * values(shape, sum(shape), torch.float32)).to(dtype)
    dy = values(shape, 7, dtype)
    hd = h.to(dev).requires_grad_(True)
    a = act8.gelu(hd)
    (dh,) = torch.autograd.grad(a, hd, dy.to(dev))
    assert a.dtype == dh.dtype == dtype
    ref, _ = gelu64(h.double())
    assert_close(a, *ref, "gelu")
    with torch.no_grad():
        a2, q, scale = torch.ops.gmdn.gelu8_fwd(hd)
        dh2, again = torch.ops.gmdn.gelu8_bwd(dy.to(dev), q, scale, True)
    want_q, want_scale = definition(h)
    assert torch.equal(q.cpu(), want_q) and torch.equal(scale.cpu(), want_scale)
    assert torch.equal(a, a2) and torch.equal(dh, dh2)
    back = (want_q.float() * want_scale.repeat_interleave(128, -1)[..., :shape[-1]]).double()
    ref, slope = gelu64(back)
    assert_close(again, *ref, "gelu again")
    g = dy.double()
    assert_close(dh, g * slope[0], g.abs() * (slope[1] + 2 * U * slope[0].abs()), "dh")


def test_gelu_tails_and_special_values():
    """Relative accuracy far into the lower tail, the identity far above, and
    NaN and infinities (GELU(-inf) is 0 times infinity: NaN by the formula)."""
    dev = _dev()
    h = torch.cat([torch.linspace(-13, 13, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 30.0, 1e4, -30.0, -1e4])])
    a = act8.gelu(h.to(dev))
    ref, _ = gelu64(h.double())
    assert_close(a, *ref, "gelu")
    a = act8.gelu(torch.tensor([math.nan, math.inf, 2.0], device=dev)).cpu()
    assert a[0].isnan() and a[1] == math.inf and abs(a[2] - 1.9544997) < 1e-6


def test_gelu_derivative_against_differences():
    """The derivative at values that the checkpoint holds exactly (a ramp of
    its steps), against central differences of the operator's forward."""
    dev = _dev()
    scale = torch.tensor(127.0 / 32) * STEP
    h = (torch.arange(-127, 128).float() * scale)[None]
    h = torch.cat([h[:, :128], h[:, 127:]], 1)  # two groups, an end of the ramp in each
    hd = h.to(dev).requires_grad_(True)
    (dh,) = torch.autograd.grad(act8.gelu(hd).sum(), hd)
    back = act8.unpack(act8.pack(hd.detach()), torch.float32)

    def slope(s):
        p, m = back + s, back - s
        return (act8.gelu(p).double() - act8.gelu(m).double()) / (p.double() - m.double())

    d1, d2 = slope(0.01), slope(0.02)
    rounding = 40 * U * (back.abs().double() + 1) / 0.01
    assert ((dh.double() - d1).abs() <= (d2 - d1).abs() + rounding).all()


def test_large_matrices_equal_their_parts():
    """Beyond 96 MB activations are loaded past the caches: the same bits."""
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(4)
    h = torch.randn(13000, 4000, generator=gen, device=dev).bfloat16()
    dy = torch.randn(13000, 4000, generator=gen, device=dev).bfloat16()

    def both(h, dy):
        a, q, s = torch.ops.gmdn.gelu8_fwd(h)
        return (a, q, s, *torch.ops.gmdn.act8_pack(h), *torch.ops.gmdn.gelu8_bwd(dy, q, s, True))

    whole = both(h, dy)
    for a in (0, 12000):
        part = both(h[a:a + 1000], dy[a:a + 1000])
        assert all(torch.equal(w[a:a + 1000], p) for w, p in zip(whole, part))


def test_deterministic_and_on_another_stream():
    dev = _dev()
    h, dy = values((3000, 1000), 1, torch.bfloat16).to(dev), values((3000, 1000), 2, torch.bfloat16).to(dev)

    def once():
        a, q, s = torch.ops.gmdn.gelu8_fwd(h)
        return (a, q, s, *torch.ops.gmdn.gelu8_bwd(dy, q, s, True))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


# ------------------------------------------------------- layers on checkpoints
# What 8 bits may move: the weights' gradients by the checkpoint's error, at
# most amax / 254 a value; with errors independent of the cotangents, a sum of
# n products moves by about sqrt(n) of them.  As a share of the gradient's
# norm: (amax / 254 / sqrt(3)) / rms, with amax / rms near 4 for normal rows:
# 0.9 % for a weight behind its own checkpoint.  Bounded at twice that, and the
# input's gradient likewise.
MOVES = 0.02


def moved(got, ref):
    return ((got.double() - ref.double()).norm() / ref.double().norm()).item()


@pytest.mark.parametrize("bias", [False, True])
def test_linear(bias):
    dev = _dev()
    x = values((4, 50, 300), 1, torch.float32).to(dev)
    w = values((200, 300), 2, torch.float32).to(dev)
    b = values((1, 200), 3, torch.float32)[0].to(dev) if bias else None
    dy = values((4, 50, 200), 4, torch.float32).to(dev)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y, ref = act8.linear(*leaves), F.linear(*leaves)
    assert torch.equal(y, ref)
    got, want = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(ref, leaves, dy)
    assert moved(got[0], want[0]) < 1e-6
    assert moved(got[1], want[1]) < MOVES
    if bias:
        assert moved(got[2], want[2]) < 1e-6
    back = act8.unpack(act8.pack(x.detach()), torch.float32)  # the weight's gradient by its definition
    exact = dy.double().reshape(-1, 200).t() @ back.double().reshape(-1, 300)
    assert moved(got[1], exact) < 1e-5


@pytest.mark.parametrize("autocast", [False, True])
def test_mlp_and_norm_mlp(autocast):
    dev = _dev()
    torch.manual_seed(0)
    x = torch.randn(3, 70, 256, device=dev, requires_grad=True)
    nw, nb = torch.randn(256, device=dev).abs().requires_grad_(True), torch.randn(256, device=dev).requires_grad_(True)
    w1 = (torch.randn(1024, 256, device=dev) / 16).requires_grad_(True)
    w2 = (torch.randn(256, 1024, device=dev) / 32).requires_grad_(True)
    dy = torch.randn(3, 70, 256, device=dev)
    tol = 2 * MOVES if autocast else MOVES  # bfloat16 products: 2^-8 a value, in six places
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        plain = F.linear(F.gelu(F.linear(x, w1)), w2)
        kept = act8.mlp(x, w1, w2)
        nplain = F.linear(F.gelu(F.linear(F.layer_norm(x, (256,), nw, nb), w1)), w2)
        nkept = act8.norm_mlp(x, nw, nb, w1, w2)
    assert kept.dtype == plain.dtype and nkept.dtype == nplain.dtype
    assert moved(kept, plain) < (5e-3 if autocast else 2e-6)
    assert moved(nkept, nplain) < (8e-3 if autocast else 2e-6)
    for got, ref, leaves in ((kept, plain, (x, w1, w2)), (nkept, nplain, (x, nw, nb, w1, w2))):
        g = torch.autograd.grad(got, leaves, dy.to(got.dtype))
        r = torch.autograd.grad(ref, leaves, dy.to(ref.dtype))
        for i, (a, b) in enumerate(zip(g, r)):
            assert a.dtype == b.dtype and a.shape == b.shape
            assert moved(a, b) < tol, i


def test_mlp_keeps_less_memory():
    """What the forward keeps: 5 and a little bytes a channel of the input
    (its own 8 bits, and the hidden layer's) beside the output."""
    dev = _dev()
    rows, d = 8192, 512
    x = torch.randn(rows, d, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w1 = torch.randn(4 * d, d, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w2 = torch.randn(d, 4 * d, device=dev, dtype=torch.bfloat16, requires_grad=True)
    act8.mlp(x, w1, w2)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = act8.mlp(x, w1, w2)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated() - before - out.numel() * 2
    assert held <= rows * d * 5 * (1 + 4 / 128) + (1 << 16), held / (rows * d)


def test_without_gradients_nothing_is_packed():
    """Under no_grad, and where nothing wants a gradient, the outputs are the
    same and no checkpoint is made."""
    dev = _dev()
    torch.manual_seed(0)
    x = torch.randn(5, 40, 128, device=dev)
    nw, w1, w2 = torch.rand(128, device=dev), torch.randn(256, 128, device=dev), torch.randn(128, 256, device=dev)

    def calls():
        return (act8.gelu(x), act8.linear(x, w1), act8.mlp(x, w1, w2), act8.norm_mlp(x, nw, None, w1, w2))

    with torch.no_grad():
        plain = calls()
    x.requires_grad_(True)
    kept = calls()
    with torch.no_grad():
        again = calls()
    for a, b, c in zip(plain, kept, again):
        assert torch.equal(a, b) and torch.equal(a, c) and b.requires_grad and not c.requires_grad
    a, q, scale = torch.ops.gmdn.gelu8_fwd(x.detach(), False)
    assert q.numel() == scale.numel() == 0 and torch.equal(a, plain[0])
    with pytest.raises(RuntimeError, match="no backward"):
        torch.ops.gmdn.gelu8_fwd(x, False)


def test_frozen_weights():
    dev = _dev()
    x = torch.randn(20, 64, device=dev, requires_grad=True)
    w1, w2 = torch.randn(96, 64, device=dev), torch.randn(64, 96, device=dev)
    (dx,) = torch.autograd.grad(act8.mlp(x, w1, w2).sum(), x)
    assert dx.shape == x.shape and torch.isfinite(dx).all()
    (dx,) = torch.autograd.grad(act8.norm_mlp(x, None, None, w1, w2).square().sum(), x)
    assert torch.isfinite(dx).all()


def test_refusals():
    dev = _dev()
    x = torch.randn(4, 300, device=dev)
    q, scale = act8.pack(x)
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        act8.pack(x.half())
    with pytest.raises(RuntimeError, match="at least one value"):
        act8.pack(x[:, :0])
    with pytest.raises(RuntimeError, match="int8"):
        act8.unpack((x, scale))
    with pytest.raises(RuntimeError, match="scale has shape"):
        act8.unpack((q, scale[:, :2]))
    with pytest.raises(RuntimeError, match="scale is on"):
        act8.unpack((q, scale.cpu()))
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        act8.unpack((q, scale), torch.float16)
    with pytest.raises(RuntimeError, match="checkpoint has shape"):
        torch.ops.gmdn.gelu8_bwd(x[:3], q, scale, False)
    with pytest.raises(RuntimeError):
        act8.gelu(torch.tensor(1.0, device=dev))
