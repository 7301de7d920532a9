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
