"""Values that are not finite reach what the recurrence takes them to and nothing else: outputs from
their token on, gradients of k and v up to it; padding behind the last token of interest
may hold anything."""
import math

import pytest
import torch
from test_decay_gpu import BF, F32, inputs

from mlx_vit_amd import chunk_decay

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "g", "s0")


def run(x):
    leaves = [x[n].detach().clone().requires_grad_(True) for n in NAMES]
    o, s = chunk_decay(*leaves)
    return dict(zip(("o", "s", "dq", "dk", "dv", "dg", "ds0"), (o.detach(), s.detach(), *torch.autograd.grad((o, s), leaves, (x["do"], x["ds"])))))


# by input: outputs that it reaches from its token on, up to it, and at it alone
REACH = {"q": ("", "dk dv", "o"), "k": ("o dq", "", "dv"), "v": ("o dq", "", "dk"), "g": ("o dq", "dk dv", ""), "do": ("", "dk dv", "dq")}


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("at", [0, 17, 45, 70, 127, 149])
def test_reach(at, D, dt):
    x = inputs(1, 150, 2, D, dt, state=True, seed=at)
    clean = run(x)
    for name, (later, earlier, own) in REACH.items():
        for bad in (math.nan, math.inf, -math.inf) if name != "g" else (math.nan,):
            y = dict(x, **{name: x[name].clone()})
            if name == "g":
                y[name][0, at, 1] = bad
            else:
                y[name][0, at, 1, D // 2 + 3] = bad     # a channel of one head
            got = run(y)
            for out in ("o", "dq", "dk", "dv"):
                assert torch.equal(got[out][:, :, 0], clean[out][:, :, 0]), (name, out)
                a, b = got[out][0, :, 1], clean[out][0, :, 1]
                # of g at t: the state before t is not read through it, nor is what is behind it in a gradient
                lo = at if out in later.split() else 0
                hi = at + 1 if out in earlier.split() and name != "g" else at if out in earlier.split() else 150
                if out in later.split():
                    assert torch.equal(a[:lo], b[:lo]), (name, bad, out)
                    assert not torch.isfinite(a[at]).all()
                elif out in earlier.split():
                    assert torch.equal(a[hi:], b[hi:]), (name, bad, out)
                    assert hi == 0 or not torch.isfinite(a[hi - 1]).all()
                elif out in own.split():
                    assert torch.equal(a[:at], b[:at]) and torch.equal(a[at + 1:], b[at + 1:]), (name, bad, out)
                    assert not torch.isfinite(a[at]).all()
                else:
                    assert torch.equal(a, b), (name, bad, out)


@pytest.mark.parametrize("dt", [BF, F32])
def test_padding_may_hold_anything(dt):
    x = inputs(2, 100, 2, 64, dt, state=True)
    y = {n: None if t is None else t.clone() for n, t in x.items()}
    for n in ("q", "k", "v"):
        y[n][1, 77:] = math.nan
    with torch.no_grad():
        a, b = (chunk_decay(*(t[n] for n in NAMES)) for t in (x, y))
    assert torch.equal(a[0][0], b[0][0]) and torch.equal(a[0][1, :77], b[0][1, :77]) and torch.equal(a[1][0], b[1][0])


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("g_too", [True, False])
def test_the_same_bits(g_too, D, dt):
    """Twenty calls on the same inputs, of several slots and chunks, with and without dg."""
    x = inputs(2, 333, 3, D, dt, state=True, seed=D)
    first = None
    for _ in range(20):
        leaves = [x[n].detach().requires_grad_(g_too or n != "g") for n in NAMES]
        o, s = chunk_decay(*leaves)
        out = [o, s, *torch.autograd.grad((o, s), [t for t in leaves if t.requires_grad], (x["do"], x["ds"]))]
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))
