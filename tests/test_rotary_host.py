"""rotary refuses numbers that are not whole, on the CPU, and takes whole ones of any integer type."""
import numpy as np
import pytest
import torch

from mlx_vit_amd import rotary

Q = torch.zeros(1, 5, 2, 32)


@pytest.mark.parametrize("kw,match", [
    (dict(grid=(2.5, 2)), "whole numbers"),
    (dict(grid=(2, 2.0)), "whole numbers"),
    (dict(grid=(2, 2), start=1.5), "whole numbers"),
    (dict(grid=(2, "2")), "whole numbers"),
    (dict(grid=(2, None)), "whole numbers"),
    (dict(grid=(2, 2), start=float("nan")), "whole numbers"),
    (dict(grid=(2, 2), sections=(8.5, 8)), "sections"),
    (dict(grid=(2, 2), sections=(8.0, 8)), "sections"),
    (dict(grid=(2, 2), sections=("8", 8)), "sections"),
    (dict(grid=(2, 2), sections=8), "sections"),
    (dict(positions=torch.arange(5), start=0.5), "start=0.5"),
])
def test_not_whole(kw, match):
    with pytest.raises(ValueError, match=match):
        rotary(Q, **kw)
    rotary_runs_to_the_device(grid=(2, 2), sections=(8, 8))     # (what is remembered of sections is of whole ones)
    with pytest.raises(ValueError, match=match):
        rotary(Q, **kw)


def rotary_runs_to_the_device(**kw):
    with pytest.raises(ValueError, match="ROCm device"):
        rotary(Q, **kw)


def test_whole_numbers_of_other_types():
    rotary_runs_to_the_device(grid=(np.int64(2), torch.tensor(3)), start=np.int32(4), sections=[np.int64(8), 8])
    rotary_runs_to_the_device(grid=[2, 3], start=True)
