"""linear_act and mlp in 64 bits with bounds on how far a computed result may be:
every bound follows the roundings, element by element.

u: half a step of the dtype, relative (bf16 2^-8, fp32 2^-24).  A product of K terms
summed in fp32 is off by at most acc * sum |a||b|, acc = (2 K + 16) 2^-24: one
rounding a term and one a sum, and (fp32) the parts of the split operands that
are left out, 3 * 2^-24 of |a||b|.  Activations: |act'| <= 1.13, |act''| <= 0.8;
the kernels' act and act' are off by at most 4e-7 (1 + |z|), a few 2^-24.
For bf16's gelu the bounds allow 4e-4 of its value and 1.5e-6, for its derivative
6e-5: what a value before the activation that is off by these products' bounds hides
anyway.  test_activations_gpu.py holds the activations themselves to a few 10^-6."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ACT = 4e-7


def act(z, name):
    if name == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(z) if name == "silu" else z


def act_grad(z, name):
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s)) if name == "silu" else torch.ones_like(z)


class Val:
    """A value and the bound on its error."""

    def __init__(self, v, e=None):
        self.v, self.e = v, torch.zeros_like(v) if e is None else e

    def __add__(self, o):
        v = self.v + o.v
        return Val(v, self.e + o.e + 2.0 ** -23 * (self.v.abs() + o.v.abs()))

    def round(self, dt):
        return Val(self.v, self.e + U[dt] * (self.v.abs() + self.e))

    @property
    def mag(self):
        return self.v.abs() + self.e

    def mm(self, o):
        K = self.v.shape[1]
        e = self.e @ o.mag + self.v.abs() @ o.e + (2 * K + 16) * 2.0 ** -24 * (self.mag @ o.mag)
        return Val(self.v @ o.v, e)

    def t(self):
        return Val(self.v.t(), self.e.t())

    def sum0(self):
        n = self.v.shape[0]
        return Val(self.v.sum(0), self.e.sum(0) + (2 * n + 16) * 2.0 ** -24 * self.mag.sum(0))

    def act(self, name, dt):
        if name is None:
            return self
        v = act(self.v, name)
        fit = 4e-4 * v.abs() + 1.5e-6 if name == "gelu" and dt == torch.bfloat16 else 0.0
        return Val(v, 1.13 * self.e + ACT * (1 + self.mag) + fit)

    def times_act_grad(self, z, name, dt):
        if name is None:
            return self
        fit = 6e-5 if name == "gelu" and dt == torch.bfloat16 else 0.0
        d = Val(act_grad(z.v, name), 0.8 * z.e + ACT * (1 + z.mag) + fit)
        return Val(self.v * d.v, self.e * d.mag + self.v.abs() * d.e + 2.0 ** -23 * self.mag * d.mag)


def _val(t, dev):
    return None if t is None else Val(t.detach().to(dev).double())


def linear_act(x, w, b, r, name, dy=None):
    """{"y", "dx", "dw", "db", "dr"}: Val each, rounded as the op rounds (gradients with dy)."""
    dt = x.dtype
    dev = x.device
    x, w, b, r, dy = (_val(t, dev) for t in (x, w, b, r, dy))
    z = x.mm(w.t())
    if b is not None:
        z = z + Val(b.v.expand(z.v.shape))
    y = z.act(name, dt)
    if r is not None:
        y = y + r
    out = {"y": y.round(dt)}
    if dy is not None:
        exact = dy if name is None else dy.times_act_grad(z.round(dt), name, dt)
        dz = exact if name is None else exact.round(dt)
        # the bias gradient sums dz before it is rounded
        out.update(dx=dz.mm(w).round(dt), dw=dz.t().mm(x).round(dt), db=exact.sum0().round(dt), dr=dy)
    return out


def mlp(x, w1, b1, w2, b2, r, name, dy=None):
    """{"y", "dx", "dw1", "db1", "dw2", "db2", "dr"}."""
    dt = x.dtype
    dev = x.device
    x, w1, b1, w2, b2, r, dy = (_val(t, dev) for t in (x, w1, b1, w2, b2, r, dy))
    z = x.mm(w1.t())
    if b1 is not None:
        z = z + Val(b1.v.expand(z.v.shape))
    h = z.act(name, dt).round(dt)
    y = h.mm(w2.t())
    if b2 is not None:
        y = y + Val(b2.v.expand(y.v.shape))
    if r is not None:
        y = y + r
    out = {"y": y.round(dt)}
    if dy is not None:
        exact = dy.mm(w2).times_act_grad(z.round(dt), name, dt)
        dz = exact.round(dt)
        # behind an activation the first bias gradient sums dz before it is rounded
        out.update(dx=dz.mm(w1).round(dt), dw1=dz.t().mm(x).round(dt), db1=(dz if name is None else exact).sum0().round(dt),
                   dw2=dy.t().mm(h).round(dt), db2=dy.sum0().round(dt), dr=dy)
    return out


def check(name, got, want):
    got = got.detach().double().to(want.v.device).reshape(want.v.shape)
    off = (got - want.v).abs() - want.e
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, f"{name}: {worst:.3e} past its bound (largest value {want.v.abs().max().item():.3e})"
