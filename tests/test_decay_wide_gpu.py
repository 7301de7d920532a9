"""chunk_decay's other paths at every head size and type, gradients too: packed sequences, shared heads,
gradients of some inputs, sequences that are shared out.  Tolerances: test_decay_gpu."""
import pytest
import torch
from test_decay_gpu import BF, F32, chain, check, inputs, near

import decay_reference as R
from mlx_vit_amd import chunk_decay

pytestmark = pytest.mark.gpu
SIZES = [32, 64, 96, 128]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("cu", [[5, 5, 70, 300], [0, 64, 128, 192, 330], [0, 1, 1, 200, 330], [7, 130], [0], [330, 330]])
def test_packed(cu, D, dt):
    x = inputs(1, 330, 2, D, dt, hk=1, state=True, n=len(cu) - 1, one=len(cu) == 4, seed=D)
    out = check(x, cu)
    for t in (out[0], *out[2:5]):     # rows of no sequence
        assert not t[0, :cu[0]].any() and not t[0, cu[-1]:].any()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("H,hq,hk,hv", [(5, 1, 5, 1), (3, 3, 1, 3)])
def test_packed_slots(H, hq, hk, hv, D, dt):
    """Sequences of several slots, odd numbers of heads (workgroups that fill no group of eight), q shared and not."""
    x = inputs(1, 900, H, D, dt, hq, hk, hv, state=True, n=3, slow=0.1, seed=H)
    check(x, [2, 520, 521, 890])


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("hq,hk,hv", [(4, 2, 2), (1, 1, 4), (2, 4, 1), (4, 4, 2), (1, 4, 4)])
def test_shared_heads(hq, hk, hv, D, dt):
    check(inputs(1, 140, 4, D, dt, hq, hk, hv, one=hq == 1, state=True, seed=D))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("T,cu", [(70, None), (700, None), (400, [0, 130, 390])])
def test_some_gradients(T, cu, D, dt):
    """Each input's gradient by itself, against 64 bits: without that of g other kernels run."""
    x = inputs(1, T, 2, D, dt, hk=1, state=True, n=1 if cu is None else 2, slow=0.2, seed=D)
    names = ("q", "k", "v", "g", "s0")
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    a = {m: None if t is None else (t / 2 if m == "g" else t.abs()) for m, t in x.items()}
    want, big = (R.backward(*(y[m] for m in names), cu, y["do"], y["ds"]) for y in (x, a))
    for i in (0, 1, 2, 4):
        some = [x[m].detach().requires_grad_(j == i) for j, m in enumerate(names)]
        got, = torch.autograd.grad(chunk_decay(*some, c), some[i], (x["do"], x["ds"]))
        near(got, want[i], big[i], dt, chain(T, D), names[i])


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", SIZES)
def test_split_over_slots(D, dt):
    """Several rows of several heads, shared out; lengths that are no multiple of a slot's."""
    check(inputs(2, 1101, 3, D, dt, state=True, slow=0.05, seed=D))


def test_past_two_to_the_31():
    """More than 2^31 elements an operand: the last tokens, whose decays forget all before, against 64 bits."""
    H, D, tail = 16, 128, 130
    T = (1 << 31) // (H * D) + 1000
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.empty(1, T, H, D, dtype=BF, device="cuda").normal_(generator=gen) for _ in range(3))
    g = torch.full((1, T, H), -0.5, device="cuda")
    g[:, T - tail] = -float("inf")
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    o, _ = chunk_decay(*leaves)
    do = torch.zeros_like(o)
    do[:, T - tail:].normal_(generator=gen)
    got = [o, *torch.autograd.grad(o, leaves, do)]
    x = [t[:, T - tail:].detach() for t in leaves]
    a = [*(t.abs() for t in x[:3]), x[3] / 2]
    d = do[:, T - tail:]
    want = [R.forward(*x)[0], *R.backward(*x, None, None, d, None)[:4]]
    big = [R.forward(*a)[0], *R.backward(*a, None, None, d.abs(), None)[:4]]
    for name, t, w, b in zip(("o", "dq", "dk", "dv", "dg"), got, want, big):
        near(t[:, T - tail:], w, b, BF, chain(T, D) if name == "dg" else chain(tail, D), name)
        if name == "dg":
            # in the 32 tokens of the border, sums over pairs behind it cancel: of at most 64 numbers in fp64 on either
            # side, each off by 64 2^-53 of the pairs' sizes, which M holds (a pair (t, s) in every M between them)
            assert bool((t[:, :T - tail].abs().amax(1).double().cpu() <= 2.0 ** -46 * b.sum(1)).all())
            assert not t[:, :T - tail - 32].any()
        elif name != "o":
            assert not t[:, :T - tail].any()
