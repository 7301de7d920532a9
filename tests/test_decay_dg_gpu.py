"""dg of chunk_decay where little of what is nearby gets through: each token's within the rounding of
its own terms.

dg_t is the sum of e^{g_{s+1} + .. + g_t'} (q_t' . k_s) (do_t' . v_s) over s < t <= t', the states
before and behind as further terms.  Tolerance: 5 (n + 2) 2^-24 of M_t, the same sum of absolute
values at the same g.  n = 2 D + 128 + T / 32 is the length of the chain of sums (as in
test_decay_gpu); a weight e^x is off by 2 (2 + |x|) 2^-24 of itself, |x| at most 100 here, which
is below n + 2.  Nothing is added for what passes elsewhere in the sequence."""
import decay_reference as R
import pytest
import torch
from test_decay_gpu import BF, DEV, F32, chain, inputs, near

from mlx_vit_amd import chunk_decay

pytestmark = pytest.mark.gpu


def case(name, D, dt, one=False):
    x = inputs(1, 200, 2, D, dt, state=True, one=one, seed=D)
    T = 200
    g = x["g"].fill_(-0.01) if not one else x["g"].fill_(-0.2)
    last = torch.zeros_like(x["do"])
    last[:, -1] = x["do"][:, -1]
    if name in ("a fast chunk, v zero", "a fast chunk"):
        g[:, 64:96] = -1.0
        x["do"], x["ds"] = last, None
        if "zero" in name:
            x["v"].zero_()
    elif name == "two fast chunks":
        g[:, 32:64] = g[:, 128:160] = -1.0
        x["do"], x["ds"] = last, None
    elif name == "the last token's loss":
        g.fill_(-0.2)
        x["do"], x["ds"] = last, None
    elif name == "the first token's value":
        g.fill_(-0.2)
        x["v"][:, 1:] = 0
        x["s0"], x["ds"] = None, None
    elif name == "fast and slow":
        g.copy_(torch.where(torch.arange(T, device=DEV) // 32 % 2 == 0, -0.01, -5.0)[None, :, None].expand_as(g))
    elif name == "fast":
        g.copy_(-15 * torch.rand(g.shape, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV))
    elif name == "early values, late loss":
        g.fill_(-0.3)
        x["v"][:, 40:] = 0
        x["do"][:, :-20] = 0
        x["ds"] = None
    return x


CASES = ["a fast chunk, v zero", "a fast chunk", "two fast chunks", "the last token's loss", "the first token's value",
         "fast and slow", "fast", "early values, late loss"]


def dg_of(x, cu=None):
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "g")]
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
    o, s = chunk_decay(*leaves, x["s0"], c)
    return torch.autograd.grad((o, s) if x["ds"] is not None else o, leaves[3],
                               (x["do"], x["ds"]) if x["ds"] is not None else x["do"])[0]


def bounds(x, cu=None):
    a = {m: None if t is None else (t.detach() if m == "g" else t.detach().abs()) for m, t in x.items()}
    return [R.backward(y["q"], y["k"], y["v"], y["g"], y["s0"], cu, y["do"], y["ds"])[3] for y in (x, a)]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("name", CASES)
def test_each_token(name, D, dt):
    x = case(name, D, dt)
    got = dg_of(x)
    want, big = bounds(x)
    near(got, want, big, dt, chain(200, D), name)


@pytest.mark.parametrize("D", [64, 128])
def test_packed_and_by_heads(D):
    """The same in the second of three packed sequences; and summed over the tokens."""
    x = case("a fast chunk", D, F32)
    cu = [0, 7, 190, 200]
    x["s0"] = torch.cat([x["s0"]] * 3)
    got = dg_of(x, cu)
    want, big = bounds(x, cu)
    near(got, want, big, F32, chain(200, D), "packed")
    x = case("", D, F32, one=True)
    got = dg_of(x)
    want, big = bounds(x)
    near(got, want, big, F32, chain(200, D), "by heads")
