"""chunk_decay's bf16 outputs are the 64-bit results rounded once, but for the few that lie next to a
border: pairs' weights and states keep 24 bits in the products.

An error e before the last rounding turns it the other way with probability |e| / step, and a step is
|y| / 256 or more: 256 |e / y|.  Errors of fp32 sums are 2^-22 of the outputs' norm here (a cut
sum of the matrix unit 2^-23, a weight, the state and the sum over both 2^-24 each), and
1 / |y| averages 4 over normal outputs down to half a step: one in 2^12.  (Weights or states of
16 bits are off by 2^-18 on average: one in 2^8 to 2^10.)"""
import decay_reference as R
import pytest
import torch
from test_decay_gpu import BF, inputs

from mlx_vit_amd import chunk_decay

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("g_too", [True, False])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_roundings(D, g_too):
    x = inputs(1, 700, 4, D, BF, state=True, slow=0.2, seed=D)
    names = ("q", "k", "v", "g", "s0")
    leaves = [x[n].requires_grad_(g_too or n != "g") for n in names]
    o, s = chunk_decay(*leaves)
    got = [o, *torch.autograd.grad((o, s), leaves[:3], (x["do"], x["ds"]))]
    want = [R.forward(*leaves)[0], *R.backward(*leaves, None, x["do"], x["ds"])[:3]]
    for name, a, b in zip(("o", "dq", "dk", "dv"), got, want):
        share = float((a.detach().cpu() != b.to(BF)).double().mean())
        assert share <= 2.0 ** -12, f"{name}: one in {1 / share:.0f} rounded the other way"
