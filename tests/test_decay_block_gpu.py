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
