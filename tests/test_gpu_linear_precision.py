"""Linear attention's results are the fp32 sums rounded once, in every type: of a sum just above the middle
between two numbers of a 16-bit type, all 24 bits decide which of the two it becomes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# Between 1 and its neighbour: the middle, and what lies above it. All three are numbers of the type, and
# their sum has 21 or 23 bits: exact in fp32, in any order.
ABOVE = {torch.float32: (2.0 ** -11, 2.0 ** -22), torch.float16: (2.0 ** -11, 2.0 ** -22), torch.bfloat16: (2.0 ** -8, 2.0 ** -20)}


def ones(x, dims=slice(None), tokens=slice(None)):
    """x with ones in those dimensions of those tokens."""
    x[:, tokens, :, dims] = 1
    return x


def terms(x, tokens=slice(None)):
    """x with the sum's terms in its first dimensions."""
    for i, y in enumerate((1.0, *ABOVE[x.dtype])):
        x[:, tokens, :, i] = y
    return x


# One chunk and several, one segment and several, waves of 32 and of 64 columns.
@pytest.mark.parametrize("dtype", list(ABOVE), ids=str)
@pytest.mark.parametrize("b, t, h, dk, dv, at", [(2, 1, 1, 32, 32, 0), (1, 30, 2, 32, 24, 5), (3, 50, 1, 64, 64, 20), (1, 300, 1, 128, 128, 70), (1030, 40, 1, 64, 64, 3)])
def test_sums_are_rounded_once(b, t, h, dk, dv, at, dtype):
    from zeno_amd.memory import linear_attention

    want = torch.tensor(1.0 + sum(ABOVE[dtype]), dtype=torch.float64).to(dtype).item()
    assert want != 1.0
    g = torch.zeros(h, device="cuda")

    def keys():
        return torch.zeros(b, t, h, dk, dtype=dtype, device="cuda")

    def values():
        return torch.zeros(b, t, h, dv, dtype=dtype, device="cuda")

    def check(y, first, last, what):
        assert (y[:, first:last] == want).all(), what
        assert not y[:, :first].any() and not y[:, last:].any(), what

    one, three = slice(at, at + 1), slice(3)
    # A key that every query from its token on meets: in the chunk's own products, then in the state.
    o, _ = linear_attention(ones(keys(), three), terms(keys(), one), ones(values(), tokens=one), g, scale=1.0)
    check(o, at, t, "o")

    def gradient(n, q, k, v, d_o):
        leaves = dict(zip("qkv", (x.requires_grad_() for x in (q, k, v))))
        return torch.autograd.grad(linear_attention(q, k, v, g, scale=1.0)[0], leaves[n], d_o)[0]

    check(gradient("q", keys(), ones(keys(), tokens=one), terms(values(), one), ones(values(), three)), at, t, "gradient of q")
    check(gradient("k", ones(keys(), tokens=one), keys(), terms(values()), ones(values(), three, one)), 0, at + 1, "gradient of k")
    check(gradient("v", ones(keys(), three, one), terms(keys()), values(), ones(values(), tokens=one)), 0, at + 1, "gradient of v")
