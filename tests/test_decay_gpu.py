"""chunk_decay and decay_step against 64-bit loops over the tokens (decay_reference).

Tolerances.  With u = 2^-24, the sum of n products is off by at most 2 n u of the sum of
their absolute values (the matrix unit may cut a sum off: a whole step of 2^-23).  A
weight e^{x} is off by at most (2 + |x|) 2 u of itself: the argument's rounding and
the exponential's; and (2 + |x|) e^{x} <= 2.5 e^{x / 2}.  So an output is off by at most

    5 (n + 2) u M + half a step of its type,   M: the same output of |inputs| at g / 2,

n the length of the chain of sums: D products for a pair, 64 pairs of a chunk, D for the
state, its own 64 and one a chunk behind it, or the slots' starts.  In bf16 the pairs' weights
and the state are cut to 16 bits, 2^-16 of M each.  dg adds what its sums
q . dq - k . dk over the sequence are off by: that of M's over all of it."""
import math

import decay_reference as R
import pytest
import torch

from mlx_vit_amd import chunk_decay, decay_step

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def inputs(B, T, H, D, dt, hq=None, hk=None, hv=None, one=False, state=False, n=None, slow=1.0, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    n = B if n is None else n
    g = -slow * torch.rand(*((H,) if one else (B, T, H)), generator=gen, device=DEV)
    return dict(q=(r(B, T, hq or H, D) * D ** -0.5).to(dt), k=(r(B, T, hk or H, D) * D ** -0.5).to(dt), v=r(B, T, hv or H, D).to(dt),
                g=g, s0=0.3 * r(n, H, D, D) if state else None, do=r(B, T, H, D).to(dt), ds=0.1 * r(n, H, D, D) if state else None)


def half(t):
    return {BF: 2.0 ** -8, F32: 2.0 ** -24}[t]


def chain(T, D):
    return 2 * D + 128 + T // 32


def near(got, want, big, dt_in, n, what, extra=0.0):
    tol = half(got.dtype) * want.abs() + (5 * (n + 2) * 2.0 ** -24 + (2.0 ** -15 if dt_in == BF and got.dtype == BF else 0.0)) * big + extra
    d = (got.detach().double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    assert bool((d <= tol + 1e-37).all()), f"{what}: off by {float(d.max())}, {float((d / (tol + 1e-37)).max())} of the tolerance"


def check(x, cu=None, grads=True):
    names = ["q", "k", "v", "g"] + (["s0"] if x["s0"] is not None else [])
    leaves = [x[n].requires_grad_(grads) for n in names]
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
    o, s = chunk_decay(x["q"], x["k"], x["v"], x["g"], x["s0"], c)
    B, T, H, D = o.shape
    n, dt = chain(T, D), x["q"].dtype
    a = {m: None if t is None else (t.detach() / 2 if m == "g" else t.detach().abs()) for m, t in x.items()}
    ro, rs = R.forward(x["q"], x["k"], x["v"], x["g"], x["s0"], cu)
    bo, bs = R.forward(a["q"], a["k"], a["v"], a["g"], a["s0"], cu)
    near(o, ro, bo, dt, n, "o")
    near(s, rs, bs, dt, n, "final state")
    if not grads:
        return o, s
    outs, cots = ((o, s), (x["do"], x["ds"])) if x["ds"] is not None else ((o,), (x["do"],))
    got = torch.autograd.grad(outs, leaves, cots)
    want = R.backward(x["q"], x["k"], x["v"], x["g"], x["s0"], cu, x["do"], x["ds"])
    big = R.backward(a["q"], a["k"], a["v"], a["g"], a["s0"], cu, a["do"], a["ds"])
    share = [H // x[m].shape[2] for m in "qkv"]
    wide = lambda t, i: t.repeat_interleave(share[i], 2)  # noqa: E731
    # what passes: q . dq and k . dk of absolute values, over the sequence
    passes = (R.heads(a["q"], H) * wide(big[0], 0)).sum(-1) + (R.heads(a["k"], H) * wide(big[1], 1)).sum(-1)
    for lo, hi, own in R.spans(T, cu, B):
        rows = slice(0, B) if cu is None else slice(0, 1)
        passes[rows, lo:hi] = passes[rows, lo:hi].sum(1, keepdim=True)
    extra = 5 * (n + 2) * 2.0 ** -24 * (passes.sum((0, 1)) if x["g"].dim() == 1 else passes)
    for name, g, w, b in zip(names, got, want, big):
        near(g, w, b, dt, n, "d" + name, extra if name == "g" else 0.0)
    return o, s, *got


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("T", [1, 2, 31, 63, 64, 65, 129, 300])
def test_lengths(dt, D, T):
    check(inputs(2, T, 2, D, dt, state=T % 2 == 1, seed=T))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("hq,hk,hv", [(4, 2, 2), (1, 1, 4), (2, 4, 1), (4, 4, 2), (1, 4, 4)])
def test_shared_heads(dt, hq, hk, hv):
    check(inputs(1, 140, 4, 32, dt, hq, hk, hv, one=hq == 1, state=True))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("slow", [0.0, 0.01, 30.0])
def test_split_over_slots(dt, D, slow):
    """Few heads: the sequence is shared out, here into uneven parts."""
    check(inputs(1, 1101, 1, D, dt, state=True, slow=slow, one=slow == 0.01))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("cu", [[0, 1, 1, 200, 330], [0, 330], [5, 5, 70, 300], [0, 64, 128, 192, 330], [0, 0, 0], [330, 330],
                                [0], [7, 130]])
def test_packed(dt, cu):
    x = inputs(1, 330, 2, 64, dt, hk=1, state=True, n=len(cu) - 1, one=len(cu) == 5)
    out = check(x, cu)
    for t in (out[0], *out[2:5]):     # rows of no sequence
        assert not t[0, :cu[0]].any() and not t[0, cu[-1]:].any()
    if x["g"].dim() == 3:
        assert not out[5][0, :cu[0]].any() and not out[5][0, cu[-1]:].any()


def test_packed_long():
    check(inputs(1, 2600, 1, 32, BF, state=True, n=4), [3, 3, 2200, 2201, 2590])


def test_more_sequences_than_a_scan_takes_at_once():
    """2^19 states of 128 x 128: the scan over their slots in two launches.  A sequence of one
    token, of values that a launch too few would not give."""
    n, D = (1 << 19) + 3, 128
    k = torch.ones(1, n, 1, D, dtype=BF, device=DEV)
    v = (torch.arange(n, device=DEV) % 251).to(BF)[None, :, None, None].expand(1, n, 1, D)
    with torch.no_grad():
        o, s = chunk_decay(k, k, v, torch.zeros(1, n, 1, device=DEV), None, torch.arange(n + 1, dtype=torch.int32, device=DEV))
    assert torch.equal(s[:, 0, 5, 7], v[0, :, 0, 0].float())
    # (128 times an integer below 251, in bf16)
    assert torch.equal(o[0, :, 0, 3], (128 * v[0, :, 0, 0].float()).to(BF))


def test_many_sequences():
    lens = [(7 * i) % 13 for i in range(1500)]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T = cu[-1] + 5
    x = inputs(1, T, 1, 32, BF, state=True, n=len(lens))
    c = torch.tensor(cu, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        o, s = chunk_decay(x["q"], x["k"], x["v"], x["g"], x["s0"], c)
        for i in (0, 1, 2, 700, 1023, 1024, 1025, 1499):
            lo, hi = cu[i], cu[i + 1]
            a, b = chunk_decay(*(x[m][:, lo:hi] for m in "qkvg"), x["s0"][i:i + 1])
            assert torch.equal(o[:, lo:hi], a) and torch.equal(s[i:i + 1], b)
        assert not o[:, cu[-1]:].any()


def test_limits_out_of_order():
    """A limit below its predecessor counts as that, one past the row as its end: nothing out of range is touched."""
    x = inputs(1, 100, 2, 32, BF, n=4)
    out = {}
    for cu in ([-5, 40, 30, 1000, 60], [0, 40, 40, 100, 100]):
        with torch.no_grad():
            out[cu[0]] = chunk_decay(x["q"], x["k"], x["v"], x["g"], None, torch.tensor(cu, dtype=torch.int32, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(*out.values()))


def test_sequences_do_not_meet():
    """Values that are not finite stay in their sequence, and behind the start of its 32 tokens; the gradients before."""
    x = inputs(1, 300, 2, 64, BF, state=True, n=3)
    cu = torch.tensor([0, 100, 230, 300], dtype=torch.int32, device=DEV)
    clean = chunk_decay(x["q"], x["k"], x["v"], x["g"], x["s0"], cu)
    for name, bad in (("q", math.inf), ("k", math.nan), ("v", -math.inf), ("g", math.nan)):
        y = {n: None if t is None else t.clone() for n, t in x.items()}
        y[name][0, 190] = bad     # the second sequence's second chunk
        leaves = [y[n].requires_grad_(True) for n in ("q", "k", "v", "g", "s0")]
        o, s = chunk_decay(*leaves, cu)
        got = torch.autograd.grad((o, s), leaves, (y["do"], y["ds"]))
        assert torch.equal(o[0, :164], clean[0][0, :164]) and torch.equal(o[0, 230:], clean[0][0, 230:])
        assert torch.equal(s[[0, 2]], clean[1][[0, 2]]) and not torch.isfinite(o[0, 190]).all()
        for t in got[:4]:
            assert torch.isfinite(t[0, :100]).all() and torch.isfinite(t[0, 230:]).all()


@pytest.mark.parametrize("dt", [BF, F32])
def test_decays_that_forget_all(dt):
    """g = -inf, the lowest value and -1000 start the state anew; g = 0 keeps all of it."""
    x = inputs(1, 150, 2, 32, dt, state=True)
    for value in (-math.inf, torch.finfo(F32).min, -1000.0):
        y = dict(x, g=x["g"].clone())
        y["g"][0, 70], y["g"][0, 128], y["g"][0, 30:40] = value, value, 0.0
        names = ("q", "k", "v", "g", "s0")
        leaves = [y[n].detach().requires_grad_(True) for n in names]
        o, s = chunk_decay(*leaves)
        got = torch.autograd.grad((o, s), leaves, (y["do"], y["ds"]))
        assert all(torch.isfinite(t).all() for t in (o, s, *got))
        a, b = chunk_decay(*(y[n][:, 70:128] for n in "qkv"), torch.where(y["g"] < -500, 0.0, y["g"])[:, 70:128])
        ro, _ = R.forward(*(y[n][:, 70:128] for n in "qkv"), y["g"][:, 70:128])
        bo, _ = R.forward(*(y[n][:, 70:128].abs() for n in "qkv"), y["g"][:, 70:128] / 2)
        near(o[:, 70:128], ro, bo, dt, chain(150, 32), "o")
        assert not got[3][0, 70].any() and not got[3][0, 128].any()


def views(t, how):
    """t's values at other strides and alignments."""
    B, T, H, D = t.shape
    if how == "heads first":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "projection":       # columns of a wider row
        w = torch.zeros(B, T, 3 * H * D + 16, dtype=t.dtype, device=t.device)
        w[..., H * D:2 * H * D] = t.flatten(2)
        return w[..., H * D:2 * H * D].unflatten(2, (H, D))
    if how == "misaligned":
        w = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
        w[1:] = t.flatten()
        return w[1:].view(t.shape)
    if how == "channels first":
        return t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
    if how == "tokens apart":
        w = torch.zeros(B, 2 * T, H, D, dtype=t.dtype, device=t.device)
        w[:, ::2] = t
        return w[:, ::2]
    return t


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("how", ["heads first", "projection", "misaligned", "channels first", "tokens apart"])
def test_strides(dt, how):
    x = inputs(2, 75, 2, 64, dt, state=True)
    names = ("q", "k", "v", "g", "s0")
    out = []
    for move in (lambda t: t, lambda t: views(t, how) if t.shape[1:] == (75, 2, 64) else t.transpose(0, 1).contiguous().transpose(0, 1)):
        leaves = [move(x[n].detach()).requires_grad_(True) for n in names]
        o, s = chunk_decay(*leaves)
        out.append((o, s, *torch.autograd.grad((o, s), leaves, (move(x["do"]), x["ds"]))))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_broadcast_inputs():
    """One token's g for all, heads by expand: their gradients are torch's sums."""
    x = inputs(2, 70, 2, 32, F32)
    k, g = x["k"][:, :, :1].clone().requires_grad_(True), x["g"][:, :1].clone().requires_grad_(True)
    o, _ = chunk_decay(x["q"], k.expand(2, 70, 2, 32), x["v"], g.expand(2, 70, 2))
    dk, dg = torch.autograd.grad(o, (k, g), x["do"])
    args = (x["q"], k.expand(2, 70, 2, 32), x["v"], g.expand(2, 70, 2), None, None, x["do"], None)
    _, wk, _, wg, _ = R.backward(*args)
    torch.testing.assert_close(dk.double().cpu(), wk.sum(2, keepdim=True), rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(dg.double().cpu(), wg.sum(1, keepdim=True), rtol=1e-4, atol=1e-3)


def test_bf16_decay():
    x = inputs(1, 70, 2, 32, BF)
    g = x["g"].bfloat16().requires_grad_(True)
    o, _ = chunk_decay(x["q"], x["k"], x["v"], g)
    h = g.detach().float().requires_grad_(True)
    p, _ = chunk_decay(x["q"], x["k"], x["v"], h)
    assert torch.equal(o, p)
    a, b = torch.autograd.grad(o, g, x["do"])[0], torch.autograd.grad(p, h, x["do"])[0]
    assert a.dtype == BF and torch.equal(a, b.bfloat16())


def test_against_differences():
    """Gradients against central differences of the fp32 kernel: h = 2^-6 makes the formula's own error
    h^2 / 6 of third derivatives (e^g's alone: at most a 2^-14th), rounding's 2^-24 / h."""
    x = inputs(1, 67, 1, 32, F32, state=True)
    names = ("q", "k", "v", "g", "s0")
    leaves = [x[n].requires_grad_(True) for n in names]
    o, s = chunk_decay(*leaves)
    grads = torch.autograd.grad((o, s), leaves, (x["do"], x["ds"]))
    gen = torch.Generator(device=DEV).manual_seed(3)
    with torch.no_grad():
        for i, (t, d) in enumerate(zip(leaves, grads)):
            e = torch.randn(t.shape, generator=gen, device=DEV)
            if names[i] == "g":
                e = e / 16
            h, f = 2.0 ** -6, []
            for sign in (1, -1):
                y = [u + sign * h * e if j == i else u for j, u in enumerate(leaves)]
                a, b = chunk_decay(*y)
                f.append((a.double() * x["do"]).sum() + (b.double() * x["ds"]).sum())
            num, want = float(f[0] - f[1]) / (2 * h), float((d.double() * e).sum())
            size = float((d.double() * e).abs().sum())
            assert abs(num - want) <= 2e-3 * size / math.sqrt(t.numel()) + 2e-3 * abs(want), names[i]


def test_some_gradients_only():
    x = inputs(1, 70, 2, 32, BF, state=True)
    full = [x[n].detach().clone().requires_grad_(True) for n in ("q", "k", "v", "g", "s0")]
    want = torch.autograd.grad(chunk_decay(*full)[0], full, x["do"])
    for i in range(5):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate(full)]
        got, = torch.autograd.grad(chunk_decay(*some)[0], some[i], x["do"])
        # without dg the state's products take two parts of it, not three: both within a bf16 step
        if i == 3 or i == 4:
            assert torch.equal(got, want[i])
        else:
            torch.testing.assert_close(got, want[i], rtol=2.0 ** -7, atol=1e-4)


def test_only_the_last_state_counts():
    x = inputs(2, 70, 2, 32, F32, state=True)
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "g", "s0")]
    _, s = chunk_decay(*leaves)
    got = torch.autograd.grad(s, leaves, x["ds"], allow_unused=True)
    want = R.backward(*leaves[:4], leaves[4], None, None, x["ds"])
    assert not got[0].any()
    for g, w in zip(got[1:], want[1:]):
        torch.testing.assert_close(g.double().cpu(), w, rtol=1e-4, atol=1e-4)


def test_in_parts():
    """A sequence in three calls, and its last tokens one by one, is the sequence in one."""
    x = inputs(2, 203, 2, 64, F32)
    with torch.no_grad():
        o, s = chunk_decay(x["q"], x["k"], x["v"], x["g"])
        state, parts = None, []
        for lo, hi in ((0, 64), (64, 101), (101, 200)):
            a, state = chunk_decay(*(x[n][:, lo:hi] for n in "qkvg"), state)
            parts.append(a)
        for t in range(200, 203):
            parts.append(decay_step(*(x[n][:, t] for n in "qkvg"), state)[:, None])
    torch.testing.assert_close(torch.cat(parts, 1), o, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(state, s, rtol=1e-5, atol=1e-5)


def test_nothing_to_do():
    for B, T in ((0, 5), (2, 0), (0, 0)):
        x = inputs(B, T, 2, 32, BF, state=True)
        leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "g", "s0")]
        o, s = chunk_decay(*leaves)
        assert o.shape == (B, T, 2, 32) and torch.equal(s, x["s0"])
        got = torch.autograd.grad((o, s), leaves, (x["do"], x["ds"]))
        assert [g.shape for g in got] == [t.shape for t in leaves] and torch.equal(got[4], x["ds"])
        o, s = chunk_decay(*leaves[:4])
        assert not s.any()
    for B, T in ((2, 0), (0, 3)):
        x = inputs(B, T, 300, 32, BF, one=True)
        g = x["g"].requires_grad_(True)
        torch.full((300,), math.nan, device=DEV)   # what freed memory holds
        dg, = torch.autograd.grad(chunk_decay(x["q"], x["k"], x["v"], g)[0], g, x["do"])
        assert dg.shape == (300,) and not dg.any()


def test_the_same_twice_and_on_another_stream():
    x = inputs(1, 1500, 3, 64, BF, hk=1, state=True, one=True)
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "g", "s0")]

    def go():
        o, s = chunk_decay(*leaves)
        return (o, s, *torch.autograd.grad((o, s), leaves, (x["do"], x["ds"])))
    first = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = go()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, go())) and all(torch.equal(a, b) for a, b in zip(first, other))


def test_captured():
    """Two graphs, forward and backward, replayed in turn with eager work between, on new values."""
    graphs = []
    for seed, (T, cu) in enumerate(((700, None), (300, [0, 64, 250]))):
        x = inputs(1, T, 2, 64, BF, hk=1, state=True, n=1 if cu is None else 2, seed=seed)
        c = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
        leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "g", "s0")]

        def go(leaves=leaves, c=c, x=x):
            o, s = chunk_decay(*leaves, c)
            return (o, s, *torch.autograd.grad((o, s), leaves, (x["do"], x["ds"])))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go()
        graphs.append((graph, out, x, go))
    for i in range(4):
        for graph, out, x, go in graphs:
            with torch.no_grad():
                x["q"].copy_(torch.randn_like(x["q"]))
                x["g"].copy_(-torch.rand_like(x["g"]))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(got, go())), i


def test_refuses_on_the_device():
    x = inputs(1, 9, 2, 32, F32, state=True)
    q = x["q"].requires_grad_(True)
    o, _ = chunk_decay(q, x["k"], x["v"], x["g"])
    d, = torch.autograd.grad(o.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    with pytest.raises(RuntimeError, match="no gradient"):
        decay_step(q[:, 0], x["k"][:, 0], x["v"][:, 0], x["g"][:, 0], x["s0"])
    with pytest.raises(ValueError, match="cu_seqlens is on"):
        chunk_decay(q, x["k"], x["v"], x["g"], None, torch.tensor([0, 9], dtype=torch.int32))
    with pytest.raises(ValueError, match="k is on"):
        chunk_decay(q, x["k"].cpu(), x["v"], x["g"])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x["k"], torch.ones_like(x["k"]))
        with pytest.raises(RuntimeError):
            chunk_decay(x["q"].detach(), dual, x["v"], x["g"])
    # a state that a graph still needs
    k = x["k"].requires_grad_(True)
    g = x["g"].requires_grad_(True)
    o, s = chunk_decay(x["q"].detach(), k, x["v"], g, x["s0"])
    with torch.no_grad():
        decay_step(*(x[n][:, 0] for n in "qkvg"), s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.sum().backward()


def test_past_two_to_the_31():
    """More than 2^31 elements an operand: the last tokens, whose decays forget all before, are as alone."""
    H, D, tail = 16, 128, 130
    T = (1 << 31) // (H * D) + 1000
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.empty(1, T, H, D, dtype=BF, device=DEV).normal_(generator=gen) for _ in range(3))
    g = torch.full((1, T, H), -0.5, device=DEV)
    g[:, T - tail] = -math.inf
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    o, s = chunk_decay(*leaves)
    do = torch.zeros_like(o)
    do[:, T - tail:].normal_(generator=gen)
    dq, dk, dv, dg = torch.autograd.grad(o, leaves, do)
    part = [t[:, T - tail:].detach().clone().requires_grad_(True) for t in leaves]
    po, ps = chunk_decay(*part)
    pd = torch.autograd.grad(po, part, do[:, T - tail:])
    near(o[:, T - tail:], po.detach().double().cpu(), 1.1 * po.detach().double().abs().cpu() + 30.0, BF, 0, "o", 2.0 ** -8 * 100)
    near(s, ps.detach().double().cpu(), ps.detach().double().abs().cpu() + 30.0, F32, 400, "state")
    for a, b in zip((dq, dk, dv), pd):
        torch.testing.assert_close(a[:, T - tail:], b, rtol=2.0 ** -6, atol=1.0)
        assert not a[:, :T - tail].any()
    torch.testing.assert_close(dg[:, T - tail + 1:], pd[3][:, 1:], rtol=1e-3, atol=10.0)


# ---------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------
def step_inputs(B, N, H, D, dt, hq=None, hk=None, hv=None, one=False, seed=0):
    x = inputs(B, 1, H, D, dt, hq, hk, hv, one, seed=seed)
    gen = torch.Generator(device=DEV).manual_seed(seed + 1)
    return [*(x[n][:, 0] for n in "qkv"), x["g"] if one else x["g"][:, 0], torch.randn(N, H, D, D, generator=gen, device=DEV)]


def check_step(q, k, v, g, state, slots=None):
    want, states = R.step(q, k, v, g, state, slots)
    a = [t.abs() for t in (q, k, v)] + [g / 2, state.abs()]
    times = 1 if slots is None else max([slots.count(n) for n in slots] or [1])
    bo, bs = R.step(*a, slots)
    at = None if slots is None else torch.tensor(slots, dtype=torch.int32, device=DEV)
    o = decay_step(q, k, v, g, state, slots=at)
    D = q.shape[-1]
    near(o, want, bo, F32, D + 4 * times, "o")
    near(state, states, bs, F32, 4 * times, "state")
    return o


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("B,H", [(1, 1), (3, 6), (5, 3)])
def test_step(dt, D, B, H):
    check_step(*step_inputs(B, B, H, D, dt, one=B == 5))


@pytest.mark.parametrize("hq,hk,hv", [(4, 2, 2), (1, 1, 4), (2, 4, 1)])
def test_step_shared_heads(hq, hk, hv):
    check_step(*step_inputs(3, 3, 4, 64, BF, hq, hk, hv))


@pytest.mark.parametrize("slots", [[2, 0, 4], [4, -1, 5], [7, 1 << 30, -(1 << 31)], [1, 1, 1], [0, 3, 0], []])
def test_step_slots(slots):
    """Slots in any order, outside the states (left out, the output zero), and the same one twice."""
    x = step_inputs(len(slots), 5, 2, 64, BF)
    before = x[4].clone()
    check_step(*x, slots)
    for n in set(range(5)) - set(slots):
        assert torch.equal(x[4][n], before[n])


def test_step_many_rows_of_few_states():
    gen = torch.Generator().manual_seed(0)
    check_step(*step_inputs(200, 40, 2, 32, F32), torch.randint(-1, 41, (200,), generator=gen).tolist())


def test_step_no_states():
    x = step_inputs(2, 0, 2, 32, BF)
    assert not check_step(*x, [0, 3]).any()


@pytest.mark.parametrize("how", ["projection", "misaligned", "channels first"])
def test_step_strides(how):
    q, k, v, g, s = step_inputs(3, 3, 2, 64, BF)
    t = s.clone()
    o = decay_step(q, k, v, g, s)
    move = lambda u: views(u[:, None], how)[:, 0]  # noqa: E731
    assert torch.equal(decay_step(move(q), move(k), move(v), g.t().contiguous().t(), t), o) and torch.equal(s, t)


def test_step_forgets_and_keeps():
    q, k, v, g, s = step_inputs(2, 2, 2, 32, F32)
    g[0], g[1] = -math.inf, 0.0
    t = s.clone()
    decay_step(q, k, v, g, s)
    assert torch.equal(s[0], v[0, :, :, None] * k[0, :, None, :])
    torch.testing.assert_close(s[1], t[1] + v[1, :, :, None] * k[1, :, None, :], rtol=2.0 ** -23, atol=2.0 ** -23)


def test_step_in_inference_mode_and_captured():
    with torch.inference_mode():
        check_step(*step_inputs(2, 2, 2, 64, BF))
    x = step_inputs(4, 6, 2, 64, BF)
    slots = torch.tensor([5, 2, 2, -1], dtype=torch.int32, device=DEV)
    twin = x[4].clone()
    decay_step(*x[:4], twin.clone(), slots=slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = decay_step(*x, slots=slots)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(decay_step(*x[:4], twin, slots=slots), o) and torch.equal(twin, x[4]), i
