"""Numbers of steps that do not fit the C structure's 32 bits are refused, not cut."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [0, -1, 101, 1 << 32, (1 << 32) + 5, 5 - (1 << 32)])
def test_refused(steps):
    from zeno_amd.optim import orthogonalize

    with pytest.raises(ValueError, match="steps"):
        orthogonalize(torch.randn(8, 9, device="cuda"), steps)
