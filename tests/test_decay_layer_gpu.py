"""DecayAttentionLayer against its formulas in 64 bits, in parts and token by token, and as a
model's mixer.

Tolerance in fp32: each stage's outputs are within 2^-16 of their sums of absolute values (the
operators' own tests bound them by far less), and a row is normed twice; 1e-4 of the
largest output covers the five stages here.  In bf16 q, k, v, o, y and the gate are rounded
to half a step, 2^-8, each: six of them add up to 2^-8 6^(1/2) = 0.01 of the output's norm."""
import pytest
import torch
import torch.nn.functional as F

from mlx_vit_amd import DecayAttentionLayer
from mlx_vit_amd.model import HybridBlock, NoPEGDNClassifier, to_bf16

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(layer, x, state=None, start=0):
    """The layer in 64 bits with torch's operations, differentiable."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in layer.named_parameters()}
    x = x.detach().double().requires_grad_(True)
    B, T, _ = x.shape
    H, D, K = layer.num_heads, layer.head_dim, layer.num_kv_heads
    q, k, v = (F.linear(x, p[n + ".weight"]).unflatten(-1, (-1, D)) for n in ("q_proj", "k_proj", "v_proj"))
    n = torch.arange(T, device=x.device) + start
    h, w = layer.grid
    at, out = 0, []
    angles = [pos.double()[:, None] * layer.base ** (-torch.arange(0, s, 2, device=x.device).double() / s)
              for pos, s in zip((n // (h * w), n // w % h, n % w), layer.sections)]

    def turn(t):
        y = []
        at = 0
        for a, s in zip(angles, layer.sections):
            c, sn, m, o = torch.cos(a)[:, None], torch.sin(a)[:, None], t[..., at:at + s // 2], t[..., at + s // 2:at + s]
            y += [m * c - o * sn, m * sn + o * c]
            at += s
        return torch.cat(y, -1)
    q, k = turn(q * layer.scale), turn(k)
    k, v = (t.repeat_interleave(H // K, 2) for t in (k, v))
    g = -torch.exp(p["A_log"]) * F.softplus(F.linear(x, p["a_proj.weight"]) + p["dt_bias"])
    s = torch.zeros(B, H, D, D, dtype=torch.float64, device=x.device) if state is None else state.double()
    for t in range(T):
        s = torch.exp(g[:, t])[..., None, None] * s + v[:, t, :, :, None] * k[:, t, :, None, :]
        out.append((s * q[:, t, :, None, :]).sum(-1))
    o = torch.stack(out, 1)
    y = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + layer.o_norm.eps) * p["o_norm.weight"]
    y = (y * torch.sigmoid(F.linear(x, p["g_proj.weight"]).unflatten(-1, (H, D)))).flatten(2)
    return F.linear(y, p["o_proj.weight"]), s, x, p


@pytest.mark.parametrize("kw", [dict(), dict(num_kv_heads=1, grid=(2, 3)), dict(head_dim=32, num_heads=4, num_kv_heads=2, sections=(16, 8, 8))])
def test_layer(kw):
    torch.manual_seed(0)
    layer = DecayAttentionLayer(48, **{**dict(num_heads=2, head_dim=64, grid=(3, 4)), **kw}).to(DEV)
    x = torch.randn(2, 70, 48, device=DEV, requires_grad=True)
    y, s = layer(x, start=7)
    dy = torch.randn_like(y)
    grads = torch.autograd.grad(y, [x, *layer.parameters()], dy)
    wy, ws, wx, p = plain(layer, x, start=7)
    want = torch.autograd.grad(wy, [wx, *p.values()], dy.double())
    for name, a, b in zip(["y", "state", "x", *p], [y, s, *grads], [wy, ws, *want]):
        assert float((a.double() - b).abs().max()) <= 1e-4 * float(b.abs().max()), name


def test_layer_in_bf16():
    torch.manual_seed(0)
    layer = to_bf16(DecayAttentionLayer(64, 2, 64, grid=(3, 4)).to(DEV))
    assert layer.A_log.dtype == layer.dt_bias.dtype == torch.float32
    x = torch.randn(2, 100, 64, device=DEV).bfloat16()
    y, s = layer(x)
    wy, ws, _, _ = plain(layer, x)
    assert y.dtype == torch.bfloat16 and s.dtype == torch.float32
    assert float((y.double() - wy).norm()) <= 0.02 * float(wy.norm())      # (and the products' two)


def test_streaming():
    """Tubelet by tubelet, then token by token, is the video at once."""
    torch.manual_seed(0)
    layer = DecayAttentionLayer(48, 2, 64, grid=(3, 4)).to(DEV)
    x = torch.randn(2, 40, 48, device=DEV)
    with torch.no_grad():
        y, s = layer(x)
        state, parts = None, []
        for lo in (0, 12, 24):
            a, state = layer(x[:, lo:lo + 12], state, start=lo)
            parts.append(a)
        for t in range(36, 40):
            parts.append(layer.step(x[:, t:t + 1], state, t))
        with pytest.raises(ValueError, match="one token"):
            layer.step(x[:, :2], state, 0)
    torch.testing.assert_close(torch.cat(parts, 1), y, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(state, s, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("time_only", [False, True])
def test_as_a_models_mixer(time_only):
    torch.manual_seed(0)
    model = NoPEGDNClassifier(img_size=32, num_frames=4, tubelet_size=(2, 16, 16), encoder_dim=64, encoder_depth=1, encoder_heads=2,
                              processor_dim=64, processor_depth=4, processor_heads=2, num_classes=5, mixer="decay",
                              gdn_temporal_only=time_only).to(DEV)
    assert model.backbone.get_block_types() == ["decay", "decay", "decay", "nope"]
    assert model.backbone.processor_blocks[0].layer.grid == ((1, 1) if time_only else (2, 2))
    video = torch.randn(2, 4, 32, 32, 3, device=DEV)
    loss = F.cross_entropy(model(video), torch.tensor([1, 3], device=DEV))
    loss.backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0, name


def test_refuses():
    for kw, match in ((dict(head_dim=48), "head_dim=48"), (dict(num_heads=6, num_kv_heads=4), "does not divide")):
        with pytest.raises(ValueError, match=match):
            DecayAttentionLayer(64, **kw)
    with pytest.raises(ValueError, match="x must be"):
        DecayAttentionLayer(64).to(DEV)(torch.zeros(2, 3, 32, device=DEV))
    with pytest.raises(ValueError, match="block_type"):
        HybridBlock(64, 2, "softmax")
    with pytest.raises(ValueError, match="mixer"):
        NoPEGDNClassifier(mixer="nope")
