"""rotary where nothing turns: sections without channels, and channels behind the axes, bit for bit."""
import pytest
import torch

from mlx_vit_amd import rotary

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda"
BITS = {BF: torch.int16, F32: torch.int32}


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [(0,), (0, 0), (0, 0, 0)])
def test_no_channels_turn(sections, interleaved, dt):
    q = torch.randn(2, 9, 3, 64, device=DEV).to(dt).requires_grad_(True)
    k = torch.randn(2, 9, 1, 64, device=DEV).to(dt)
    for where in (dict(grid=(2, 3)), dict(positions=torch.arange(9, device=DEV).expand(len(sections), 9))):
        y, z = rotary(q, k, sections=sections, interleaved=interleaved, **where)
        d, = torch.autograd.grad(y, q, y)
        assert torch.equal(y, q) and torch.equal(z, k) and torch.equal(d, y)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_channels_behind_the_axes_keep_their_bits(interleaved, dt):
    """A zero's sign among them."""
    q = torch.randn(1, 5, 2, 64, device=DEV).to(dt)
    q[..., 33:50:3], q[..., 34:50:3] = -0.0, 0.0
    y = rotary(q, grid=(2, 2), start=9, sections=(16, 8, 8), interleaved=interleaved)
    assert torch.equal(y[..., 32:].contiguous().view(BITS[dt]), q[..., 32:].contiguous().view(BITS[dt]))
