"""linear_act and mlp against 64-bit formulas with a bound for every element
(linear_reference): sizes that end inside a tile, rows of every alignment, one
row to several tiles, each activation, dtype and optional operand; strided and
expanded operands, frozen inputs, no rows, graph replays, finite differences."""
import pytest
import torch

import linear_reference as L

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}

# M, K, N
SIZES = [(1, 8, 1), (1, 384, 174), (3, 5, 7), (17, 33, 19), (64, 40, 130), (65, 8, 8), (65, 7, 9), (128, 64, 128),
         (129, 100, 257), (131, 31, 33), (200, 384, 520), (300, 772, 395), (257, 520, 136), (70, 1536, 384),
         # forwards in tiles of 64 x 64 (bf16 alone or both; few steps and many), the largest in pieces
         (700, 33, 200), (2100, 41, 130), (3000, 96, 7), (2060, 130, 136), (2050, 1501, 130), (9, 600, 5000),
         (8, 70, 8200)]


def _mk(seed, *shape, dt, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dt).to(DEV)


def _inputs(M, K, N, dt, bias=True, res=True, seed=0):
    return (_mk(seed, M, K, dt=dt), _mk(seed + 1, N, K, dt=dt, scale=K ** -0.5),
            _mk(seed + 2, N, dt=dt, scale=0.1) if bias else None, _mk(seed + 3, M, N, dt=dt) if res else None,
            _mk(seed + 4, M, N, dt=dt))


def _leaves(*ts):
    for t in ts:
        if t is not None:
            t.requires_grad_(True)
    return [t for t in ts if t is not None]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_act_forward_and_gradients(size, dtype):
    from mlx_vit_amd import linear_act
    M, K, N = size
    i = SIZES.index(size)
    for act, bias, res in ((None, True, False), ("gelu", i % 3 != 0, i % 2 == 0), ("silu", i % 3 != 1, i % 2 == 1)):
        print(size, dtype, act, bias, res, flush=True)
        x, w, b, r, dy = _inputs(M, K, N, DT[dtype], bias, res, seed=10 * i)
        want = L.linear_act(x, w, b, r, act, dy)
        with torch.no_grad():
            plain = linear_act(x, w, b, r, act)
        L.check("y without gradients", plain, want["y"])
        leaves = _leaves(x, w, b, r)
        y = linear_act(x, w, b, r, act)
        assert torch.equal(y, plain)
        names = ["dx", "dw"] + ["db"] * (b is not None) + ["dr"] * (r is not None)
        for n, g, leaf in zip(names, torch.autograd.grad(y, leaves, dy), leaves):
            assert g.shape == leaf.shape and g.dtype == leaf.dtype
            L.check(n, g, want[n])


# M, K, hidden
MLP_SIZES = [(1, 64, 128), (5, 9, 27), (64, 96, 384), (66, 72, 144), (130, 67, 201), (300, 384, 1536), (257, 128, 520)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", MLP_SIZES, ids=str)
def test_mlp_forward_and_gradients(size, dtype):
    from mlx_vit_amd import mlp
    M, K, N = size
    i, dt = MLP_SIZES.index(size), DT[dtype]
    for act, res in (("gelu", i % 2 == 0), ("silu", i % 2 == 1), (None, True)):
        print(size, dtype, act, res, flush=True)
        x, w1, b1, _, _ = _inputs(M, K, N, dt, i % 4 != 3, False, seed=100 + 10 * i)
        _, w2, b2, r, dy = _inputs(M, N, K, dt, i % 4 != 2, res, seed=500 + 10 * i)
        want = L.mlp(x, w1, b1, w2, b2, r, act, dy)
        with torch.no_grad():
            plain = mlp(x, w1, b1, w2, b2, r, act)
        leaves = _leaves(x, w1, b1, w2, b2, r)
        y = mlp(x, w1, b1, w2, b2, r, act)
        assert torch.equal(y, plain)
        L.check("y", y, want["y"])
        names = ["dx", "dw1"] + ["db1"] * (b1 is not None) + ["dw2"] + ["db2"] * (b2 is not None) + ["dr"] * (r is not None)
        for n, g in zip(names, torch.autograd.grad(y, leaves, dy)):
            L.check(n, g, want[n])


# Shapes for each tile size the launches choose from (by the number of tiles), ending inside one:
# bf16 256 x 256 (K from 512), 128 x 128, 64 x 64; fp32 128 x 128, 128 x 64, 64 x 64
TILED = [(6210, 2049, 520, "bf16", "gelu"), (5000, 3300, 72, "bf16", "silu"), (6200, 2560, 640, "bf16", None),
         (2100, 1030, 200, "bf16", None), (3000, 2100, 50, "bf16", "gelu"),
         (5000, 3300, 40, "fp32", "gelu"), (4200, 1030, 72, "fp32", None), (700, 513, 136, "fp32", "silu")]


@pytest.mark.parametrize("M,N,K,dtype,act", TILED)
def test_every_tile_size(M, N, K, dtype, act):
    from mlx_vit_amd import linear_act, mlp
    dt = DT[dtype]
    x, w, b, r, dy = _inputs(M, K, N, dt, seed=200)
    want = L.linear_act(x, w, b, r, act, dy)
    leaves = _leaves(x, w, b, r)
    y = linear_act(x, w, b, r, act)
    L.check("y", y, want["y"])
    for n, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves[:3], dy)):
        L.check(n, g, want[n])
    # as a block's second map: dgrad over K' = K with the derivative of the first's activation, N wide
    x, w1, b1, _, _ = _inputs(M, 24, N, dt, True, False, seed=210)
    _, w2, b2, _, dy = _inputs(M, N, K, dt, True, False, seed=220)
    want = L.mlp(x, w1, b1, w2, b2, None, "gelu", dy)
    leaves = _leaves(x, w1, b1, w2, b2)
    y = mlp(x, w1, b1, w2, b2)
    L.check("y", y, want["y"])
    for n, g in zip(("dx", "dw1", "db1", "dw2", "db2"), torch.autograd.grad(y, leaves, dy)):
        L.check(n, g, want[n])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strided_operands(dtype):
    """Column slices, a transposed weight, a 3-d input, rows behind an offset of one
    element, an expanded cotangent."""
    from mlx_vit_amd import linear_act
    dt = DT[dtype]
    B, T, K, N = 3, 37, 72, 56
    wide = _mk(1, B, T, 3 * K + 1, dt=dt)
    wt = _mk(2, K, N, dt=dt, scale=K ** -0.5)
    b, r = _mk(3, 2 * N, dt=dt)[::2], _mk(4, B, T, 2 * N, dt=dt)[..., N:]
    for at in (0, 1, K):
        x = wide[..., at:at + K]
        want = L.linear_act(x.reshape(-1, K), wt.t(), b, r.reshape(-1, N), "gelu", torch.ones(B * T, N, dtype=dt))
        leaves = [t.detach().requires_grad_(True) for t in (x, wt, b, r)]
        y = linear_act(leaves[0], leaves[1].t(), leaves[2], leaves[3], "gelu")
        assert y.shape == (B, T, N)
        L.check("y", y.reshape(-1, N), want["y"])
        dx, dwt, db, dr = torch.autograd.grad(y.sum(), leaves)     # its cotangent is one expanded element
        L.check("dx", dx.reshape(-1, K), want["dx"])
        L.check("dw", dwt.t(), want["dw"])
        L.check("db", db, want["db"])
        L.check("dr", dr.reshape(-1, N), want["dr"])
    one = _mk(5, 1, K, dt=dt).expand(80, K)                        # rows at a stride of zero
    L.check("expanded rows", linear_act(one, wt.t()), L.linear_act(one, wt.t(), None, None, None)["y"])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_shared_operands(dtype):
    """x as its own residual, and one weight for both maps: the gradients add up."""
    from mlx_vit_amd import mlp
    dt = DT[dtype]
    M, K = 90, 64
    x, w, b, _, dy = _inputs(M, K, K, dt, True, False, seed=30)
    want = L.mlp(x, w, b, w, b, x, "gelu", dy)
    leaves = _leaves(x, w, b)
    y = mlp(x, w, b, w, b, x, "gelu")
    L.check("y", y, want["y"])
    for n, g in zip(("x", "w", "b"), torch.autograd.grad(y, leaves, dy)):
        parts = {"x": ("dx", "dr"), "w": ("dw1", "dw2"), "b": ("db1", "db2")}[n]
        L.check(n, g, (want[parts[0]] + want[parts[1]]).round(dt))


def test_frozen_inputs_get_no_gradient():
    from mlx_vit_amd import linear_act, mlp
    x, w, b, r, dy = _inputs(70, 64, 96, torch.bfloat16)
    want = L.linear_act(x, w, b, r, "silu", dy)
    for i, n in enumerate(("dx", "dw", "db", "dr")):
        ts = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w, b, r))]
        linear_act(*ts, "silu").backward(dy)
        assert [t.grad is not None for t in ts] == [i == j for j in range(4)]
        L.check(n, ts[i].grad, want[n])
    x, w1, b1, _, _ = _inputs(70, 64, 96, torch.bfloat16, seed=1)
    _, w2, b2, r, dy = _inputs(70, 96, 64, torch.bfloat16, seed=2)
    want = L.mlp(x, w1, b1, w2, b2, r, "gelu", dy)
    for i, n in enumerate(("dx", "dw1", "db1", "dw2", "db2", "dr")):
        ts = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w1, b1, w2, b2, r))]
        mlp(*ts, "gelu").backward(dy)
        assert [t.grad is not None for t in ts] == [i == j for j in range(6)]
        L.check(n, ts[i].grad, want[n])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_no_rows(dtype):
    from mlx_vit_amd import linear_act, mlp
    dt = DT[dtype]
    x, w1, b1, _, _ = _inputs(0, 16, 24, dt, True, False)
    _, w2, b2, r, dy = _inputs(0, 24, 16, dt)
    leaves = _leaves(x, w1, b1, w2, b2, r)
    for y, ls in ((mlp(x, w1, b1, w2, b2, r), leaves), (linear_act(x, w1, b1, None, "gelu"), leaves[:3])):
        assert y.shape[0] == 0
        for g, t in zip(torch.autograd.grad(y.sum(), ls), ls):
            assert g.shape == t.shape and not g.any()


def test_non_finite_values_stay_in_their_rows():
    """A NaN or infinite row of x makes that row of y non-finite and no other, also
    where the row ends inside a tile of the contracted index."""
    from mlx_vit_amd import linear_act
    for dt in (torch.bfloat16, torch.float32):
        for M, K, N in ((70, 36, 40), (200, 136, 130), (9, 20, 24)):
            x, w, b, r, _ = _inputs(M, K, N, dt, seed=7)
            clean = linear_act(x, w, b, r, "gelu")
            x[3, K - 1] = float("nan")
            x[5, 0] = float("inf")
            y = linear_act(x, w, b, r, "gelu")
            rows = torch.ones(M, dtype=torch.bool, device=DEV)
            rows[3] = rows[5] = False
            assert y[3].isnan().all() and not y[5].isfinite().all()
            assert torch.equal(y[rows], clean[rows])


def test_gelu_over_its_range():
    """Values from -40 to 40 through the epilogue and its derivative (K = 1)."""
    from mlx_vit_amd import linear_act
    for dt in (torch.bfloat16, torch.float32):
        for act in ("gelu", "silu"):
            x = torch.linspace(-40, 40, 4001, device=DEV).to(dt).unsqueeze(1).requires_grad_(True)
            w = torch.ones(1, 1, dtype=dt, device=DEV)
            want = L.linear_act(x, w, None, None, act, torch.ones(4001, 1, dtype=dt))
            y = linear_act(x, w, None, None, act)
            L.check("y", y, want["y"])
            L.check("dx", torch.autograd.grad(y.sum(), x)[0], want["dx"])


def test_gradients_against_differences():
    """Central differences of sum(y dy) along a random direction of each input, fp32.
    Truncation: h^2 / 6 times a third derivative of order the slope itself (h = 1/64:
    4e-5); rounding: each y is off by at most 2^-24 of its terms' sum, some 2^-20,
    and 90 x 48 of them of random sign add up to 66 * 2^-20 / (2 h) = 2e-3, against
    slopes of order 66: 1e-3 relative to the largest slope covers both."""
    from mlx_vit_amd import mlp
    M, K, N = 90, 48, 80
    x, w1, b1, _, _ = _inputs(M, K, N, torch.float32, True, False, seed=40)
    _, w2, b2, r, dy = _inputs(M, N, K, torch.float32, seed=41)
    ts = _leaves(x, w1, b1, w2, b2, r)
    grads = torch.autograd.grad(mlp(*ts), ts, dy)
    h = 2.0 ** -6
    got, want = [], []
    with torch.no_grad():
        for i, t in enumerate(ts):
            d = _mk(50 + i, *t.shape, dt=torch.float32)
            d = d / d.norm() * 8
            f = [(mlp(*[s + e * h * d if j == i else s for j, s in enumerate(ts)]).double() * dy.double()).sum().item()
                 for e in (1, -1)]
            want.append((f[0] - f[1]) / (2 * h))
            got.append((grads[i].double() * d.double()).sum().item())
    print("slopes", got, want, flush=True)
    scale = max(abs(v) for v in want)
    assert all(abs(a - b) <= 1e-3 * max(scale, 66.0) for a, b in zip(got, want))


def test_second_derivative_is_refused():
    from mlx_vit_amd import linear_act
    x, w, b, r, dy = _inputs(5, 16, 8, torch.float32)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(linear_act(x, w, b, r, "gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_graph_replays(dtype):
    """A captured inference pass and a captured training pass replay on new inputs,
    the program's own eager work between the replays."""
    from mlx_vit_amd import mlp
    dt = DT[dtype]
    for M in (9, 150):
        x, w1, b1, _, _ = _inputs(M, 64, 132, dt, True, False, seed=60)
        _, w2, b2, r, dy = _inputs(M, 132, 64, dt, seed=61)
        ts = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2, r)]

        def step():
            y = mlp(*ts)
            return [y.detach(), *torch.autograd.grad(y, ts, dy)]

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for k in range(3):
            with torch.no_grad():
                ts[0].copy_(_mk(70 + k, M, 64, dt=dt))
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, step()):
                assert torch.equal(a, b)


def test_graph_replays_of_large_tiles():
    """The tiles of 256 x 256 take more LDS than a kernel gets by default."""
    from mlx_vit_amd import linear_act
    x, w, b, r, _ = _inputs(6200, 640, 2560, torch.bfloat16, seed=65)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = linear_act(x, w, b, r, "gelu")
    for k in range(3):
        x.copy_(_mk(75 + k, 6200, 640, dt=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, linear_act(x, w, b, r, "gelu"))


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad
    from mlx_vit_amd import linear_act, mlp
    x, w, b, _, _ = _inputs(9, 16, 16, torch.float32)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: linear_act(d, w, b), lambda: mlp(d, w, b, w, b)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("M", [5, 4100])
def test_values_past_fp16(M, act):
    """z of +-3 10^5: the activation is z or nothing there, its derivative 1 or 0."""
    from mlx_vit_amd import linear_act
    x = torch.full((M, 8), 300000.0, dtype=torch.bfloat16, device=DEV)
    x[1::2] = -x[1::2]
    w = torch.eye(8, dtype=torch.bfloat16, device=DEV)
    dy = _mk(90, M, 8, dt=torch.bfloat16)
    leaves = _leaves(x, w)
    y = linear_act(x, w, activation=act)
    assert torch.equal(y, x.clamp(min=0))
    dx, dw = torch.autograd.grad(y, leaves, dy)
    # gelu's derivative is off by at most 6e-5 (the sum in linear_reference: the fit's 2.92e-5 and 1.83e-5 between the
    # true one's value where the fit ends and here), silu's by nothing here; dw's rounding, and its sum by 2^-20 of its terms
    d = 6e-5 if act == "gelu" else 0.0
    with torch.no_grad():
        dz = torch.where(x > 0, dy, 0).double()
        assert ((dx.double() - dz).abs() <= d * dy.double().abs()).all()
        want, size = dz.t() @ x.double(), 3e5 * dy.double().abs().sum(0).unsqueeze(1)
        assert ((dw.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -20 + d) * size).all()


def test_other_stream():
    from mlx_vit_amd import mlp
    x, w1, b1, _, _ = _inputs(300, 64, 128, torch.bfloat16, True, False, seed=80)
    _, w2, b2, r, dy = _inputs(300, 128, 64, torch.bfloat16, seed=81)
    ref = mlp(x, w1, b1, w2, b2, r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = mlp(x, w1, b1, w2, b2, r)
    s.synchronize()
    assert torch.equal(y, ref)


def test_results_repeat_bit_for_bit():
    from mlx_vit_amd import mlp
    for dt in (torch.bfloat16, torch.float32):
        x, w1, b1, _, _ = _inputs(1000, 96, 200, dt, True, False, seed=90)
        _, w2, b2, r, dy = _inputs(1000, 200, 96, dt, seed=91)
        ts = _leaves(x, w1, b1, w2, b2, r)
        a, b = (torch.autograd.grad(mlp(*ts), ts, dy) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_blocks_mlp_as_one_operator():
    """A block with ``set_fused_mlp`` against itself without: the separate modules round
    the value before the activation and each map's result too.  And the cases that
    keep the modules: dropout in training, a hook."""
    from mlx_vit_amd import model as M
    for dt in (torch.bfloat16, torch.float32):
        torch.manual_seed(0)
        blk = M.NoPEViTBlock(64, 2, 4.0, dropout=0.1).to(DEV).to(dt).eval()
        x = _mk(1, 2, 50, 64, dt=dt).requires_grad_(True)
        ps = [x, *blk.parameters()]
        outs = []
        for on in (False, True):
            M.set_fused_mlp(blk, on)
            y = blk(x)
            outs.append([y, *torch.autograd.grad(y.float().square().sum(), ps)])
        # relative to each tensor's norm: a few roundings of u, at random
        tol = 8 * torch.finfo(dt).eps
        for a, b in zip(*outs):
            assert (a.double() - b.double()).norm() <= tol * b.double().norm()
        calls = []
        import mlx_vit_amd.model as mod
        real, mod.mlp = mod.mlp, lambda *a, **k: calls.append(1) or real(*a, **k)
        try:
            blk(x)
            assert calls == [1]
            blk.train()
            blk(x)
            h = blk.eval().mlp[0].register_forward_hook(lambda *a: None)
            blk(x)
            h.remove()
            assert calls == [1]
            blk(x)
            assert calls == [1, 1]
        finally:
            mod.mlp = real


def test_tracing_is_refused():
    from mlx_vit_amd import linear_act, mlp
    x, w, b, _, _ = _inputs(9, 16, 16, torch.float32)
    for f in (lambda t: linear_act(t, w, b), lambda t: mlp(t, w, b, w, b)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_offsets_past_32_bits(dtype):
    """More than 2^31 elements in y, z, dy and dz: the first and the last rows, and what sums over all."""
    from mlx_vit_amd import linear_act
    M, K, N = 131142, 16, 16392
    dt = DT[dtype]
    x, w = _mk(300, M, K, dt=dt), _mk(301, N, K, dt=dt, scale=0.25)
    row = _mk(302, N, dt=dt)
    leaves = _leaves(x, w)
    y = linear_act(x, w, activation="silu")
    dx, dw = torch.autograd.grad(y, leaves, row.expand(M, N))
    with torch.no_grad():
        for rows in (slice(0, 70), slice(M - 70, M)):
            want = L.linear_act(x[rows], w, None, None, "silu", row.expand(70, N).contiguous())
            L.check("y", y[rows], want["y"])
            L.check("dx", dx[rows], want["dx"])
        # the last 8 columns' dw: half a step for dz's rounding and one for its own, and the sum's 2 M 2^-24
        z = x.double() @ w[-8:].double().t()
        sg = torch.sigmoid(z)
        dz = row[-8:].double() * sg * (1 + z * (1 - sg))
        want, size = dz.t() @ x.double(), dz.abs().t() @ x.double().abs()
        tol = (2 * M + 16) * 2.0 ** -24 * size + torch.finfo(dt).eps * (size + want.abs())
        assert ((dw[-8:].double() - want).abs() <= tol).all()


class _Scale(torch.nn.Identity):
    def forward(self, x):
        return 0.5 * x


def _drop_paths():
    """What a block's drop_path may be, by name, as it comes out of ``block.eval()``."""
    from mlx_vit_amd.model import DropPath
    train = DropPath(0.5)
    hooked, own = torch.nn.Identity(), DropPath(0.3)
    hooked.register_forward_hook(lambda m, args, out: 0.25 * out)
    own.forward = lambda x: 2 * x
    return {"identity": torch.nn.Identity(), "evaluated": DropPath(0.5), "training": train, "a scale": _Scale(),
            "a linear map": torch.nn.Linear(64, 64), "hooked": hooked, "its own forward": own, "never": DropPath(0.0)}


@pytest.mark.parametrize("name", list(_drop_paths()))
@pytest.mark.parametrize("kind", ["NoPEViTBlock", "HybridBlock"])
def test_blocks_mlp_and_what_follows_it(kind, name):
    """A block's drop_path sees the MLP's result with ``set_fused_mlp`` as without: stochastic depth that is on in an
    evaluated block, another module in its place, hooks.  Tolerances as in test_blocks_mlp_as_one_operator."""
    from mlx_vit_amd import model as M
    torch.manual_seed(0)
    blk = M.NoPEViTBlock(64, 2) if kind == "NoPEViTBlock" else M.HybridBlock(64, 2, "nope")
    blk.drop_path = _drop_paths()[name]
    blk = blk.to(DEV).eval()
    if name in ("training", "never"):
        blk.drop_path.train()
    x = _mk(1, 16, 10, 64, dt=torch.float32)
    outs = []
    for on in (False, True):
        M.set_fused_mlp(blk, on)
        torch.manual_seed(1)
        y = blk(x)
        outs.append(y if kind == "NoPEViTBlock" else y[0])
    a, b = (o.detach().double() for o in outs)
    for i in range(16):
        assert (a[i] - b[i]).norm() <= 8 * torch.finfo(torch.float32).eps * a[i].norm(), i


class _NoAttention(torch.nn.Module):
    """(The library's attention has no second derivative of its own.)"""

    def forward(self, x, mask=None):
        return torch.sin(x)


def test_blocks_mlp_under_transforms():
    """torch.func's transforms take the modules: one block over several inputs, per-sample gradients, a Hessian."""
    from mlx_vit_amd import model as M
    torch.manual_seed(0)
    blk = M.NoPEViTBlock(16, 2).to(DEV).eval()
    blk.attn = _NoAttention()
    x = _mk(1, 3, 2, 5, 16, dt=torch.float32)
    outs = []
    for on in (False, True):
        M.set_fused_mlp(blk, on)
        outs.append((torch.func.vmap(blk)(x), torch.func.vmap(torch.func.grad(lambda t: blk(t).square().sum()))(x),
                     torch.func.vjp(blk, x[0])[1](x[1])[0],
                     torch.func.hessian(lambda t: blk(t[None, None]).square().sum())(x[0, 0, 0])))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    calls = []
    real, M.mlp = M.mlp, lambda *a, **k: calls.append(1) or real(*a, **k)
    try:
        blk(x[0])
        assert calls == [1]
    finally:
        M.mlp = real


# M, K, hidden, outputs: outputs that are no multiple of 8 (dy is copied), few from many columns and the reverse, one,
# and two whose first map's gradient takes tiles of 256 x 256 by one of the widths and smaller ones by the other
OTHER_WIDTHS = [(131, 300, 520, 7), (70, 8, 72, 513), (257, 33, 64, 1), (1, 24, 40, 130), (9, 130, 96, 600),
                (300, 96, 384, 200), (64, 1000, 24, 16), (6200, 24, 2560, 640), (6200, 640, 2560, 24)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", OTHER_WIDTHS, ids=str)
def test_mlp_of_other_output_width(size, dtype):
    from mlx_vit_amd import mlp
    M, K, N, O = size
    i, dt = OTHER_WIDTHS.index(size), DT[dtype]
    for act, bias, res in (("gelu", True, i % 2 == 0), ("silu", i % 2 == 1, True), (None, True, False))[:1 if M > 6000 else 3]:
        print(size, dtype, act, bias, res, flush=True)
        x, w1, b1, _, _ = _inputs(M, K, N, dt, bias, False, seed=400 + 10 * i)
        _, w2, b2, r, dy = _inputs(M, N, O, dt, True, res, seed=600 + 10 * i)
        want = L.mlp(x, w1, b1, w2, b2, r, act, dy)
        with torch.no_grad():
            plain = mlp(x, w1, b1, w2, b2, r, act)
        leaves = _leaves(x, w1, b1, w2, b2, r)
        y = mlp(x, w1, b1, w2, b2, r, act)
        assert y.shape == (M, O) and torch.equal(y, plain)
        L.check("y", y, want["y"])
        names = ["dx", "dw1"] + ["db1"] * (b1 is not None) + ["dw2", "db2"] + ["dr"] * (r is not None)
        for n, g, leaf in zip(names, torch.autograd.grad(y, leaves, dy), leaves):
            assert g.shape == leaf.shape
            L.check(n, g, want[n])


def test_blocks_mlp_with_frozen_weights(monkeypatch):
    """Where a bias is trained and its weight is not, the modules run: no weight's gradient is formed in vain."""
    from mlx_vit_amd import model as M
    torch.manual_seed(0)
    blk = M.NoPEViTBlock(64, 2).to(DEV)
    M.set_fused_mlp(blk)
    x = _mk(1, 2, 50, 64, dt=torch.float32)
    calls = []
    real = M.mlp
    monkeypatch.setattr(M, "mlp", lambda *a, **k: calls.append(1) or real(*a, **k))
    for frozen, fused in (((), True), ((0, 3), False), ((0,), False), ((3,), False)):
        blk.requires_grad_(True)
        for i in frozen:
            blk.mlp[i].weight.requires_grad_(False)
        blk.zero_grad()
        calls.clear()
        blk(x).square().sum().backward()
        assert bool(calls) == fused
        assert all((p.grad is not None) == p.requires_grad for p in blk.mlp.parameters())
        with torch.no_grad():
            calls.clear()
            blk(x)
            assert calls
    blk.mlp.requires_grad_(False)
    calls.clear()
    blk(x).square().sum().backward()
    assert calls
