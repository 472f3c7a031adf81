"""One training step of an LM on the residual stream's operators, and of the same LM on
torch's modules, beside it in float64 on the CPU.  The operators round where the modules
round or later (a stream's norm from the unrounded sum, logits not at all), and their sums are
float32 as the modules' are: no parameter's gradient may be further from float64 than twice
what the modules' is.  In float32 the head's products are in 'ieee'; its pieces in 'tf32' are
2^-18 of a value off each, a few of them beside the modules' error: 2e-5 of the norm more.  A
loss, which is one number, may be right by chance on either side: in bfloat16 half a step
of it is allowed."""
import pytest
import torch
import torch.nn as nn

from gmdn_amd import ops  # noqa: F401
from gmdn_amd import scan
from gmdn_amd.mixer import LM
from test_gpu_lm_stream import _dev, _pair, _step

pytestmark = pytest.mark.gpu
B, F = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,autocast,precision", [(F, False, "ieee"), (F, False, "tf32"), (F, True, "tf32"), (B, False, "tf32")])
def test_step_beside_float64(dtype, autocast, precision):
    dev = _dev()
    ours, theirs = _pair(dev, dtype)
    exact = LM(300, 128, 2, 2, "delta")
    for blk in exact.blocks:
        blk.mixer = nn.Linear(128, 128, bias=False)
    exact.load_state_dict({k: v.float().cpu() for k, v in theirs.state_dict().items()})
    for m in exact.modules():
        if isinstance(m, nn.RMSNorm):
            m.eps = torch.finfo(F).eps  # theirs; by default float64's here
    exact = exact.double()
    idx = torch.randint(300, (2, 129), generator=torch.Generator().manual_seed(1))
    x = exact._hidden(idx[:, :-1])
    loss = nn.functional.cross_entropy(exact.lm_head(x).flatten(0, 1), idx[:, 1:].flatten())
    loss.backward()
    before = scan.get_precision()
    scan.set_precision(precision)
    try:
        la, ga = _step(ours, idx.to(dev), autocast)
    finally:
        scan.set_precision(before)
    lb, gb = _step(theirs, idx.to(dev), autocast)
    more = 2e-5 if dtype == F and not autocast and precision == "tf32" else 2.0 ** -21
    loss, half = float(loss.detach()), 2.0 ** -9 if dtype == B or autocast else 0.0
    assert abs(float(la) - loss) <= 2 * abs(float(lb) - loss) + (more + half) * loss
    for n, p in exact.named_parameters():
        a, b = ((g[n].double().cpu() - p.grad).norm() / p.grad.norm() for g in (ga, gb))
        assert a <= 2 * b + more, (n, float(a), float(b))
