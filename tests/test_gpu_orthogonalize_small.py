"""Orthogonalised updates at the lower end of fp32's range."""
import pytest
import torch

from tests.policy_reference import assert_near, orthogonalize as reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [1e-7, 1e-36, 1e-38, 1.5e-45])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_a_zero_matrix_stays_zero_whatever_eps(dtype, eps):
    from zeno_amd.optim import orthogonalize

    assert not orthogonalize(torch.zeros(2, 70, 40, dtype=dtype, device="cuda"), eps=eps).any()


@pytest.mark.parametrize("size", [1e-30, 1e-36, 1e-41])
def test_small_values(size):
    """Down to numbers below fp32's normal range, which keep few digits themselves."""
    from zeno_amd.optim import orthogonalize

    x = torch.randn(40, 60, generator=torch.Generator().manual_seed(1)) * size
    got, want = orthogonalize(x.cuda(), eps=1e-44), reference(x, eps=float(torch.tensor(1e-44)))
    assert_near(got, want, 3e-5 + 2.0 ** -24)
