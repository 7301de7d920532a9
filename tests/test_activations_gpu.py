"""The activations of linear_act and mlp value by value: a map of one column with
weight one, so that its result is the activation of x (exact in every dtype used) and
its input's gradient the derivative, against 64 bits.  A result may be off by its own
rounding, half the distance of two neighbours at that value, and by the few
roundings of fp32 arithmetic before it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BITS = {torch.bfloat16: 8, torch.float32: 24}


def _half_step(v, dt):
    """Half the distance between two values of dt at |v| (normal numbers)."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -126))) - BITS[dt])


def _points(lo, hi):
    """Every bf16 value between lo and hi of at least 2^-10: exact in fp16 too."""
    x = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.cat([-x.flip(0), x])
    x = x[x.isfinite() & (x.float().abs() >= 2.0 ** -10)]
    return x[(x.float() >= lo) & (x.float() <= hi)].to(DEV)


def _phi(z):
    """Phi by erfc: (1 + erf) / 2 is zero below -8.3 in 64 bits, where Phi is 1 / z^2 of gelu'."""
    return 0.5 * torch.special.erfc(-z * math.sqrt(0.5))


def _terms(z):
    """Phi(-|z|) + |z| phi(z): gelu' below zero is their difference."""
    a = z.abs()
    return _phi(-a) + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)


def _gelu(z):
    return z * _phi(z)


def _gelu_grad(z):
    return _phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _map(x, N, act, dt):
    """y and dx of N columns that all hold the activation of x; dy is one in the first."""
    from mlx_vit_amd import linear_act
    x = x.to(dt).unsqueeze(1).requires_grad_(True)
    y = linear_act(x, torch.ones(N, 1, dtype=dt, device=DEV), activation=act)
    dy = torch.zeros_like(y)
    dy[:, 0] = 1
    return y.detach(), torch.autograd.grad(y, x, dy)[0].squeeze(1)


def _mlp(x, act, dt):
    """The same through an MLP of hidden width one: the derivative in a product's epilogue."""
    from mlx_vit_amd import mlp
    x = x.to(dt).unsqueeze(1).requires_grad_(True)
    one = torch.ones(1, 1, dtype=dt, device=DEV)
    y = mlp(x, one, None, one, None, activation=act)
    return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0].squeeze(1)


def _check(name, got, want, tol):
    off = (got.double() - want).abs() - tol
    i = off.argmax().item()
    assert (off <= 0).all(), f"{name}: {int((off > 0).sum())} of {off.numel()} off, worst {got.reshape(-1)[i].item()} for " \
                             f"{want.reshape(-1)[i].item()}"


@pytest.mark.parametrize("N", [1, 72, 0], ids=["pieces", "tiles", "mlp"])
def test_gelu_in_bf16(N):
    """The fit for e^{z^2/2} Phi(-|z|) is within 1e-5 of its value up to 6 (1e-11 of gelu beyond), e within z^2 / 2
    times three roundings of its argument and its own: 3.4e-6 at 6.  Of the derivative's terms 1.6e-6 and, in z^2,
    2e-7 cover the same."""
    x = _points(-12, 40)
    y, dx = _map(x, N, "gelu", torch.bfloat16) if N else _mlp(x, "gelu", torch.bfloat16)
    z = x.double()
    want = _gelu(z)
    _check("gelu", y, want.unsqueeze(1).expand(y.shape),
           (_half_step(want, torch.bfloat16) + 1.5e-5 * want.abs() + 2e-11).unsqueeze(1).expand(y.shape))
    want = _gelu_grad(z)
    _check("gelu'", dx, want, _half_step(want, torch.bfloat16) + (4e-6 + 2e-7 * z * z) * _terms(z) + 2.0 ** -24 * (z > 0))


def _dense(lo, hi, n=50001):
    """fp32 values between lo and hi, none of them zero."""
    return torch.linspace(lo, hi, n, dtype=torch.float64).to(DEV).float().add(2.0 ** -12)


@pytest.mark.parametrize("N", [1, 72, 0], ids=["pieces", "tiles", "mlp"])
def test_gelu_in_fp32(N):
    """Phi(-a), a = |z|, relative: the fit 8.4e-9 up to 2.5 and e^(a - 2.5) of it beyond; e by three roundings of its
    argument, 3 2^-24 a^2 / 2 = 9e-8 a^2, and its own 2^-23; w = c / (1 + c) by 2 2^-23 (the sum, the reciprocal's 2^-23,
    the product), of which the polynomial P(w) passes on w P' / P, at most 0.8 a times; its roundings, each 2^-24 of a
    partial value, 2.75 (a + 1) P 2^-24 in all; the product with e 2^-24: 3.5e-7 + 3.6e-7 a + 9e-8 a^2 + the fit.  Above zero
    1 - x adds 2^-24, and gelu's product one more."""
    x = _dense(-12, 40)
    y, dx = _map(x, N, "gelu", torch.float32) if N else _mlp(x, "gelu", torch.float32)
    z = x.double()
    a = z.abs()
    rel = 3.5e-7 + 3.6e-7 * a + 9e-8 * a * a + 8.4e-9 * torch.exp((a - 2.5).clamp(min=0, max=10))
    want = _gelu(z)
    tol = torch.where(z < 0, (rel + 2.0 ** -24) * want.abs(), z * (rel * _phi(-a) + 2.0 ** -23))
    _check("gelu", y, want.unsqueeze(1).expand(y.shape), tol.unsqueeze(1).expand(y.shape))
    _check("gelu'", dx, _gelu_grad(z), (rel + 2.0 ** -24) * _terms(z) + 2.0 ** -24 * (z > 0))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N", [1, 72, 0], ids=["pieces", "tiles", "mlp"])
def test_silu(N, dtype):
    """fp32: sigma is an exponential within 2^-23 of its value, a sum, a quotient of 2^-24 each, and one product:
    2.5 2^-23.  bf16's argument of exp2 adds |z| 2^-24 twice, its exp2 and reciprocal 2^-23 each.  The derivative is
    sigma (1 + z (1 - sigma)), where 1 - sigma is off by 2^-24 and what sigma is."""
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = _points(-60, 60) if dtype == "bf16" else _dense(-80, 80)
    y, dx = _map(x, N, "silu", dt) if N else _mlp(x, "silu", dt)
    z = x.double()
    s = torch.special.expit(z)
    rel = 2.0 ** -22 if dtype == "fp32" else 2.0 ** -21 + 2.0 ** -23 * z.abs()
    own = (lambda v: _half_step(v, dt)) if dtype == "bf16" else lambda v: 0.0
    want = z * s
    tol = own(want) + (rel + 2.0 ** -24) * want.abs()
    _check("silu", y, want.unsqueeze(1).expand(y.shape), tol.unsqueeze(1).expand(y.shape))
    t = torch.special.expit(-z)
    want = s * (1 + z * t)
    tol = s * ((1 + z.abs() * t) * (rel + 2.0 ** -22) + z.abs() * (2.0 ** -23 + rel * s))
    _check("silu'", dx, want, own(want) + tol)
