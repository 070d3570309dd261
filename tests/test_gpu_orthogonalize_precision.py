"""Orthogonalised updates of bfloat16 matrices are off by no more than their own rounding and what
fp32 products leave, whatever the matrix: dense, with few rows that are not zero, diagonal."""
import pytest
import torch

from tests.policy_reference import orthogonalize as reference

pytestmark = pytest.mark.gpu

# Operands of 22 bits and fp32 sums: 3 * 2^-21 a step, grown by at most 3.4445 in each later one, would be
# 3e-4 if all of it were aligned with the smallest singular directions; a tenth covers these matrices.
PRODUCTS = 3e-5


def matrix(kind, dtype):
    r = torch.Generator().manual_seed(3)
    if kind == "diagonal":
        x = torch.zeros(256, 300)
        x[0, 0], x[1, 1], x[2, 2] = 0.9, 0.37, 0.22
    elif kind == "identity":
        x = 0.013 * torch.eye(256)
    elif isinstance(kind, int):  # rows that are not zero, as a table's gradient has
        x = torch.zeros(256, 512)
        x[7:7 + 5 * kind:5] = torch.randn(kind, 512, generator=r)
    else:
        x = torch.randn(*kind, generator=r)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("kind", [(256, 1024), (512, 512), (1024, 1024), (700, 257), 1, 4, 37, "diagonal", "identity"], ids=str)
def test_no_more_than_the_rounding_of_the_result(kind, dtype):
    """With e the exact value and d the error before rounding, |round(e + d) - e| is at most
    |round(e) - e| + 2 |d| for every value, as the distance to the nearest number changes by |d| at most."""
    from zeno_amd.optim import orthogonalize

    x = matrix(kind, dtype)
    want = reference(x)
    rounding = float((want.to(dtype).double() - want).norm())
    error = float((orthogonalize(x.cuda()).double().cpu() - want).norm())
    assert error <= rounding + 2 * PRODUCTS * float(want.norm()), (error / float(want.norm()), rounding / float(want.norm()))
