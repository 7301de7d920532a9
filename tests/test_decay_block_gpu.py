"""A decay block that goes on from a state: in parts as at once, with the tokens' numbers."""
import pytest
import torch

from mlx_vit_amd import DecayAttentionLayer
from mlx_vit_amd.model import HybridBlock


@pytest.mark.gpu
@pytest.mark.parametrize("cuts", [(0, 24, 36), (0, 1, 36), (0, 7, 19, 36)])
def test_block_in_parts(cuts):
    """fp32; 1e-4 of what is near 1 covers each stage's sums, as for the layer."""
    torch.manual_seed(0)
    block = HybridBlock(48, 2, "decay", 64, grid=(2, 3)).cuda().eval()
    x = torch.randn(2, 36, 48, device="cuda")
    with torch.no_grad():
        y, s = block(x)
        state, parts = None, []
        for lo, hi in zip(cuts, cuts[1:]):
            a, state = block(x[:, lo:hi], state=state, start=lo)
            parts.append(a)
    torch.testing.assert_close(torch.cat(parts, 1), y, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(state, s, rtol=1e-4, atol=1e-4)


def test_a_state_needs_the_first_tokens_number():
    x, state = torch.zeros(1, 6, 64), torch.zeros(1, 2, 32, 32)
    with pytest.raises(ValueError, match="without start"):
        HybridBlock(64, 2, "decay", grid=(2, 3))(x, state=state)
    with pytest.raises(ValueError, match="without start"):
        DecayAttentionLayer(64, 2, 32)(x, state)


@pytest.mark.gpu
def test_blocks_without_positions_leave_start():
    torch.manual_seed(0)
    x, state = torch.randn(1, 6, 64, device="cuda"), 0.1 * torch.randn(1, 2, 32, 32, device="cuda")
    for kind, kw in (("gdn", dict(state=state)), ("nope", {})):
        block = HybridBlock(64, 2, kind).cuda().eval()
        with torch.no_grad():
            assert all(torch.equal(a, b) if a is not None else b is None for a, b in zip(block(x, **kw), block(x, start=5, **kw)))


@pytest.mark.gpu
@pytest.mark.parametrize("time_only", [False, True])
def test_block_against_64_bits(time_only):
    """The whole block, and of a scan over time alone each location's own sequence, with its gradients: 2e-4 of the
    largest, the layer's 1e-4 and as much for the norms and the MLP."""
    from test_decay_layer_gpu import plain
    torch.manual_seed(0)
    block = HybridBlock(48, 2, "decay", 32, spatial_tokens=6 if time_only else None, gdn_temporal_only=time_only, grid=(2, 3)).cuda()
    x = torch.randn(2, 30, 48, device="cuda", requires_grad=True)
    y, _ = block(x)
    dy = torch.randn_like(y)
    names = ["x", *(n for n, _ in block.named_parameters())]
    got = [y, *torch.autograd.grad(y, [x, *block.parameters()], dy)]
    p = {n: t.detach().double().requires_grad_(True) for n, t in block.named_parameters()}
    wx = x.detach().double().requires_grad_(True)
    n1 = torch.nn.functional.layer_norm(wx, (48,), p["norm1.weight"], p["norm1.bias"], 1e-6)
    rows = n1.reshape(2, 5, 6, 48).transpose(1, 2).reshape(12, 5, 48) if time_only else n1
    # (the layer in 64 bits has leaves of its own: its gradients are asked for with what reaches its output)
    ly, _, lx, lp = plain(block.layer, rows.detach())
    at = ly.detach().requires_grad_(True)
    mixed = at.reshape(2, 6, 5, 48).transpose(1, 2).reshape(2, 30, 48) if time_only else at
    h = wx + mixed
    n2 = torch.nn.functional.layer_norm(h, (48,), p["norm2.weight"], p["norm2.bias"], 1e-6)
    mlp = block.mlp
    ps = [p["mlp." + n] for n, _ in mlp.named_parameters()]
    f = torch.nn.functional
    wy = h + f.linear(f.gelu(f.linear(n2, ps[0], ps[1])), ps[2], ps[3])
    leaves = [wx, at, p["norm2.weight"], p["norm2.bias"], *ps]
    gx, ga, g2w, g2b, *gp = torch.autograd.grad(wy, leaves, dy.double(), retain_graph=True)
    gl = torch.autograd.grad(ly, [lx, *lp.values()], ga)
    more = torch.autograd.grad(rows, [wx, p["norm1.weight"], p["norm1.bias"]], gl[0])
    want = {"x": gx + more[0], "norm1.weight": more[1], "norm1.bias": more[2], "norm2.weight": g2w, "norm2.bias": g2b,
            **{"layer." + n: t for n, t in zip(lp, gl[1:])}, **{"mlp." + n: t for (n, _), t in zip(mlp.named_parameters(), gp)}}
    for name, a, b in zip(["y", *names], got, [wy, *(want[n] for n in names)]):
        assert float((a.double() - b).abs().max()) <= 2e-4 * float(b.abs().max()), name


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(sections=(64,)), dict(sections=(32, 32))])
def test_streams_at_different_times(kw):
    """Rows with numbers and states of their own, in a prompt and token by token, as each alone."""
    torch.manual_seed(0)
    layer = DecayAttentionLayer(48, 2, 64, grid=(3, 4), **kw).cuda()
    x, starts = torch.randn(3, 20, 48, device="cuda"), [0, 31, 12 * 700 + 5]
    at = torch.tensor(starts, device="cuda")
    near = dict(rtol=1e-4, atol=1e-4)
    with torch.no_grad():
        state = 0.1 * torch.randn(5, 2, 64, 64, device="cuda")
        slots = [4, 0, 2]
        y, s = layer(x[:, :18], state[slots], start=at)
        pool = state.clone()
        pool[slots] = s
        tails = [layer.step(x[:, t:t + 1], pool, (at + t).int(), torch.tensor(slots, dtype=torch.int32, device="cuda")) for t in (18, 19)]
        for b, n in enumerate(starts):
            one, last = layer(x[b:b + 1, :18], state[slots[b]:slots[b] + 1], start=n)
            torch.testing.assert_close(y[b:b + 1], one, **near)
            for i, t in enumerate((18, 19)):
                torch.testing.assert_close(tails[i][b:b + 1], layer.step(x[b:b + 1, t:t + 1], last, n + t), **near)
            torch.testing.assert_close(pool[slots[b]:slots[b] + 1], last, **near)
        assert torch.equal(pool[[1, 3]], state[[1, 3]])


@pytest.mark.gpu
def test_a_captured_step_goes_on():
    """Its numbers are read anew with every replay."""
    torch.manual_seed(0)
    layer = DecayAttentionLayer(48, 2, 64, grid=(3, 4)).cuda()
    x, at = torch.randn(2, 1, 48, device="cuda"), torch.tensor([3, 90], device="cuda")
    state = 0.1 * torch.randn(2, 2, 64, 64, device="cuda")
    twin = state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(x, state.clone(), at)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.step(x, state, at)
    for i in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        # (the projections' products may be made by another of torch's kernels in a graph)
        torch.testing.assert_close(y, layer.step(x, twin, torch.tensor([3 + i, 90 + i], device="cuda")), rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(state, twin, rtol=1e-5, atol=1e-5)
        at += 1


def test_start_is_refused():
    layer = DecayAttentionLayer(64, 2, 32)
    x, state = torch.zeros(2, 6, 64), torch.zeros(2, 2, 32, 32)
    for start in (torch.zeros(3, dtype=torch.int64), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2)):
        with pytest.raises(ValueError, match="start must be"):
            layer(x, state, start)
    for start in (1.5, torch.tensor(1.5)):
        with pytest.raises(ValueError, match="whole numbers"):
            layer(x, state, start)
