"""rotary against 64-bit rotations.

Tolerance: cos and sin are within 2^-23 of theirs (an angle's fraction of a turn is rounded
to fp32, 2 pi 2^-25 of a radian, and sincospif's own 2 steps), products and sum within
2^-24 each: 2^-21 (|x| + |y|) covers them; and half a step of the output's type.  The
angles of both sides are fp64 products of a position p and a frequency, rounded, at most
1, so 2^-52 |p| off each (of 2^36, the farthest here, 1.5e-5): 2^-51 |p| (|x| + |y|)."""
import math

import pytest
import torch

from mlx_vit_amd import chunk_decay, rotary

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def turned(t, positions, sections, base=10000.0, interleaved=False, back=False):
    """(values, what they may be off before rounding) in 64 bits; positions (axes, B, T)."""
    t = t.detach().double().cpu()
    y, size, at = t.clone(), torch.zeros_like(t), 0
    for p, s in zip(positions.double().cpu(), sections):
        for i in range(s // 2):
            a, b = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + s // 2 + i)
            angle = (p * base ** (-2 * i / s))[:, :, None] * (-1 if back else 1)
            c, n = torch.cos(angle), torch.sin(angle)
            y[..., a], y[..., b] = t[..., a] * c - t[..., b] * n, t[..., a] * n + t[..., b] * c
            size[..., a] = size[..., b] = (t[..., a].abs() + t[..., b].abs()) * (2.0 ** -21 + 2.0 ** -51 * p.abs())[:, :, None]
        at += s
    return y, size


def near(got, want, what):
    y, size = want
    tol = {BF: 2.0 ** -8, F32: 2.0 ** -24}[got.dtype] * y.abs() + size
    d = (got.detach().double().cpu() - y).abs()
    assert bool((d <= tol).all()), f"{what}: off by {float(d.max())}"


def check(B, T, hq, hk, D, dt, sections, positions=None, grid=None, start=0, interleaved=False, base=10000.0, move=lambda t: t):
    gen = torch.Generator(device=DEV).manual_seed(T)
    r = lambda h: torch.randn(B, T, h, D, generator=gen, device=DEV).to(dt)  # noqa: E731
    q, k, dq, dk = move(r(hq)).requires_grad_(True), move(r(hk)).requires_grad_(True), move(r(hq)), move(r(hk))
    y = rotary(q, k, positions, grid=grid, start=start, sections=sections, base=base, interleaved=interleaved)
    g = torch.autograd.grad(y, (q, k), (dq, dk))
    if grid:
        n = torch.arange(T) + start
        p = torch.stack([n // (grid[0] * grid[1]), n // grid[1] % grid[0], n % grid[1]])[:len(sections)]
    else:
        p = positions.cpu().reshape(-1, positions.shape[-2] if positions.dim() == 3 else 1, T)
    if p.dim() == 2:
        p = p[:, None]
    p = p.expand(len(sections), B, T)
    for name, got, x, back in (("q", y[0], q, False), ("k", y[1], k, False), ("dq", g[0], dq, True), ("dk", g[1], dk, True)):
        near(got, turned(x, p, sections, base, interleaved, back), name)
        assert got.is_contiguous()
        rest = sum(sections)
        assert torch.equal(got[..., rest:], x[..., rest:])
    with torch.no_grad():
        kw = dict(positions=positions, grid=grid, start=start, sections=sections, base=base, interleaved=interleaved)
        assert torch.equal(rotary(q, **kw), y[0])
    return y


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,sections", [(64, (16, 24, 24)), (128, (128,)), (96, (24, 36, 36)), (32, (8, 12)), (6, (2, 0, 4)), (64, (64,)),
                                        (2, (2,)), (256, (128, 64, 64)), (10, (4, 4)), (80, (16, 32)), (128, (64, 64))])
def test_sections(dt, interleaved, D, sections):
    p = torch.stack([torch.arange(37, device=DEV) // (a + 1) for a in range(len(sections))])
    check(2, 37, 3, 1, D, dt, sections, p, interleaved=interleaved)
    check(2, 37, 1, 2, D, dt, sections, grid=(3, 5), start=11, interleaved=interleaved)


@pytest.mark.parametrize("T", [1, 2, 196, 1571])
def test_lengths(T):
    check(3, T, 6, 6, 64, BF, (16, 24, 24), grid=(14, 14), start=196 * 1000)


@pytest.mark.parametrize("start", [(1 << 24) + 1, (1 << 31) - 20, (1 << 40) + 3])
def test_far(start):
    """Angles of far positions, numbers past 32 bits among them."""
    check(1, 40, 2, 2, 64, F32, (32, 16, 16), grid=(3, 5), start=start)
    check(1, 40, 2, 2, 64, F32, (64,), torch.arange(40, device=DEV) + min(start, 1 << 30))


@pytest.mark.parametrize("kind", ["int32", "int64", "float32", "batch", "strided", "negative"])
def test_positions(kind):
    p = torch.randint(0, 5000, (2, 3, 29), generator=torch.Generator().manual_seed(0)).to(DEV)
    if kind in ("int32", "int64"):
        p = p[:, 0].to(getattr(torch, kind))
    elif kind == "float32":
        p = p[:, 0].float() + 0.25
    elif kind == "strided":
        p = p.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    elif kind == "negative":
        p = -p
    check(3, 29, 2, 2, 64, BF, (24, 40), p)
    check(3, 29, 2, 2, 64, F32, (24, 40), p, interleaved=True, base=500.0)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("how", ["heads first", "projection", "misaligned", "channels first", "odd rows"])
def test_strides(dt, interleaved, how):
    def move(t):
        B, T, H, D = t.shape
        if how == "heads first":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if how == "channels first":
            return t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
        if how == "misaligned":
            w = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
            w[1:] = t.flatten()
            return w[1:].view(t.shape)
        w = torch.zeros(B, T, 3 * H * D + (7 if how == "odd rows" else 0), dtype=t.dtype, device=t.device)
        w[..., H * D:2 * H * D] = t.flatten(2)
        return w[..., H * D:2 * H * D].unflatten(2, (H, D))
    check(2, 21, 3, 3, 64, dt, (16, 24, 24), grid=(2, 3), interleaved=interleaved, move=move)


def test_channels_behind_the_axes_are_copied():
    """Whatever they hold, and whatever their neighbours hold."""
    q = torch.randn(1, 3, 2, 64, device=DEV)
    q[..., 40], q[..., 51], q[..., 63] = math.inf, math.nan, -math.inf
    y = rotary(q, positions=torch.arange(3, device=DEV), sections=(32,))
    assert torch.equal(y[..., 32:].isnan(), q[..., 32:].isnan()) and torch.equal(y[..., 32:].nan_to_num(7), q[..., 32:].nan_to_num(7))
    assert torch.isfinite(y[..., :32]).all()


def test_relative():
    """Scores depend on differences of positions only."""
    q, k = torch.randn(1, 1, 1, 64, device=DEV), torch.randn(1, 1, 1, 64, device=DEV)
    at = lambda n: torch.tensor([n], device=DEV)  # noqa: E731
    score = [float((rotary(q, positions=at(m)).double() * rotary(k, positions=at(n)).double()).sum())
             for m, n in ((5, 2), (1003, 1000), (3 + (1 << 20), 1 << 20))]
    assert max(score) - min(score) <= 64 * 2.0 ** -19


def test_nothing_and_one_gradient():
    for B, T in ((0, 4), (2, 0)):
        q = torch.zeros(B, T, 2, 32, device=DEV, requires_grad=True)
        y, z = rotary(q, q, grid=(2, 2))
        assert y.shape == z.shape == q.shape and torch.autograd.grad(y, q, y)[0].shape == q.shape
    q, k = torch.randn(1, 9, 2, 32, device=DEV), torch.randn(1, 9, 1, 32, device=DEV, requires_grad=True)
    y, z = rotary(q, k, grid=(3, 3), sections=(8, 12, 12))
    d = torch.randn_like(z)
    g, = torch.autograd.grad(z, k, d)
    near(g, turned(d, torch.stack([torch.arange(9) // 9, torch.arange(9) // 3 % 3, torch.arange(9) % 3])[:, None], (8, 12, 12), back=True), "dk")


def test_refuses_on_the_device():
    q = torch.randn(1, 4, 2, 32, device=DEV, requires_grad=True)
    y = rotary(q, grid=(2, 2))
    d, = torch.autograd.grad(y.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    with pytest.raises(ValueError, match="positions is on"):
        rotary(q, positions=torch.arange(4))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            rotary(torch.autograd.forward_ad.make_dual(q.detach(), torch.ones_like(q)), grid=(2, 2))


def test_captured_and_on_another_stream():
    q = torch.randn(2, 50, 3, 64, device=DEV).to(BF).requires_grad_(True)
    k = torch.randn(2, 50, 1, 64, device=DEV).to(BF).requires_grad_(True)
    p = torch.arange(50, device=DEV)[None].repeat(3, 1)

    def go():
        y = rotary(q, k, p, sections=(16, 24, 24))
        return (*y, *torch.autograd.grad(y, (q, k), y))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = go()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, go()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    for i in range(3):
        p.add_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, go())), i


def test_past_two_to_the_31():
    T = (1 << 31) // (16 * 128) + 100
    q = torch.empty(1, T, 16, 128, dtype=BF, device=DEV).normal_()
    y = rotary(q, positions=torch.arange(T, device=DEV))
    for lo in (0, T - 40):
        near(y[:, lo:lo + 40], turned(q[:, lo:lo + 40], (torch.arange(40) + lo)[None, None], (128,)), lo)


def test_more_tokens_than_a_launch_takes():
    """2^24 tokens of 256 single channels: two launches.  One row for all of them, off its pieces' alignment."""
    T, D = (1 << 24) + 3, 256
    row = torch.randn(D + 1, device=DEV).to(BF)[1:]
    y = rotary(row.expand(1, T, 1, D), grid=(64, 64), sections=(128, 64, 64))
    for lo in (0, (1 << 24) - 2):
        n = torch.arange(5) + lo
        at = torch.stack([n // 4096, n // 64 % 64, n % 64])[:, None]
        near(y[:, lo:lo + 5], turned(row.expand(1, 5, 1, D), at, (128, 64, 64)), lo)


def test_together():
    """Positions, then the attention over a clip, then a token at a time: one rotation and one recurrence over it all."""
    from mlx_vit_amd import decay_step
    B, T, H, D = 2, 150, 2, 64
    q, k, v = (torch.randn(B, T, H, D, device=DEV) * D ** -0.5 for _ in range(3))
    g = -torch.rand(B, T, H, device=DEV)
    how = dict(grid=(3, 4), sections=(16, 24, 24))
    with torch.no_grad():
        whole, last = chunk_decay(*rotary(q, k, **how), v, g)
        o, s = chunk_decay(*rotary(q[:, :147], k[:, :147], **how), v[:, :147], g[:, :147])
        for t in range(147, T):
            a, b = rotary(q[:, t:t + 1], k[:, t:t + 1], start=t, **how)
            o = torch.cat([o, decay_step(a[:, 0], b[:, 0], v[:, t], g[:, t], s)[:, None]], 1)
    torch.testing.assert_close(o, whole, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(s, last, rtol=1e-5, atol=1e-5)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    grads = torch.autograd.grad(chunk_decay(*rotary(q, k, **how), v, g)[0].square().sum(), leaves)
    assert all(torch.isfinite(t).all() and t.any() for t in grads)
