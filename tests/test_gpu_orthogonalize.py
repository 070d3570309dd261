"""Newton-Schulz orthogonalisation on the GPU against its definition in 64 bits."""
import pytest
import torch

from tests.policy_reference import HALF_ULP, assert_near, orthogonalize as reference

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]

# Largest relative error (2-norm) of a result before its own rounding. A relative error d of X
# grows by at most 3.4445 a step (the largest slope of the step's polynomial), 485 in five. With
# operands of 22 bits and fp32 sums, each of the three products of a step is off by at most about
# 2^-21, and errors of later steps grow less: 3 * 2^-21 * (1 + 3.4 + ... + 3.4^4) = 3e-4 if all
# were aligned with the smallest singular directions, which hold a share of the norm that the
# growth itself brings up to 1; a tenth of it covers random matrices. With one part of 11 bits
# (bfloat16 from 256 rows on) X is still carried in 32 bits and a product is off by 2^-12 averaged
# over at least 256 terms: 3 * 2^-12 * 485 / 16 / 10 = 2.2e-3, with the result's own rounding.
TWO_PARTS, ONE_PART = 3e-5, 2.2e-3


def tolerance(x):
    one = x.dtype == torch.bfloat16 and min(x.shape[-2:]) >= 256
    return HALF_ULP[x.dtype] + (ONE_PART if one else TWO_PARTS)


def matrices(shape, dtype, seed, rank=0):
    """Gaussian, or with `rank` strong directions over noise, as a momentum has."""
    r = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=r)
    if rank:
        x = 0.05 * x + torch.randn(*shape[:-1], rank, generator=r) @ torch.randn(*shape[:-2], rank, shape[-1], generator=r)
    return (x * 1e-3).to(dtype)


# every tile size and slice count: tiny, tall and wide, odd, several matrices, one to many tiles
SHAPES = [(1, 1), (1, 50), (3, 2), (64, 64), (65, 63), (17, 1191), (700, 40), (3, 130, 257), (2, 2, 33, 100), (300, 300), (257, 1000), (513, 512),
          (16, 256, 128), (1100, 1030)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(shape, dtype):
    from zeno_amd.optim import orthogonalize

    x = matrices(shape, dtype, seed=sum(shape), rank=4 if min(shape[-2:]) > 8 else 0)
    got = orthogonalize(x.cuda())
    assert got.dtype == dtype and got.shape == x.shape
    assert_near(got, reference(x), tolerance(x))


@pytest.mark.parametrize("shape", [(2048, 2048), (4200, 300), (512, 8192)], ids=str)
def test_large(shape):
    """The large tiles; the definition's products on the GPU, in float64."""
    from zeno_amd.optim import orthogonalize

    x = matrices(shape, torch.bfloat16, seed=1, rank=8)
    y = x.cuda().double()
    y = y.T.contiguous() if shape[0] > shape[1] else y
    y = y / (y.norm() + 1e-7)
    for _ in range(5):
        s = y @ y.T.contiguous()
        y = 3.4445 * y + (-4.7750 * s + 2.0315 * (s @ s)) @ y
    assert_near(orthogonalize(x.cuda()), y.T if shape[0] > shape[1] else y, tolerance(x))


def test_largest_tiles():
    """Enough tiles of 256 squared for every product: four matrices of 2048 x 2304."""
    from zeno_amd.optim import orthogonalize

    x = matrices((4, 2048, 2304), torch.bfloat16, seed=2, rank=8).cuda()
    y = x.double()
    y = y / (torch.linalg.matrix_norm(y)[:, None, None] + 1e-7)
    for _ in range(5):
        s = y @ y.mT.contiguous()
        y = 3.4445 * y + (-4.7750 * s + 2.0315 * (s @ s)) @ y
    assert_near(orthogonalize(x), y, tolerance(x))


def test_singular_values_come_near_one():
    from zeno_amd.optim import orthogonalize

    s = torch.linalg.svdvals(orthogonalize(matrices((200, 300), torch.float32, 3).cuda()).double().cpu())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides_and_places(dtype):
    """Transposed, sliced and expanded views in; out given, transposed, misaligned, in place."""
    from zeno_amd.optim import orthogonalize

    x = matrices((2, 70, 90), dtype, 4).cuda()
    want = orthogonalize(x)
    assert torch.equal(orthogonalize(x.mT).mT, want)
    assert torch.equal(orthogonalize(x.mT.contiguous().mT), want)
    assert torch.equal(orthogonalize(x[:1].expand(3, 70, 90))[2], want[0])
    wide = torch.zeros(2, 70, 101, dtype=dtype, device="cuda")
    wide[:, :, 3:93] = x
    assert torch.equal(orthogonalize(wide[:, :, 3:93], out=wide[:, :, 3:93]), want)
    assert not wide[:, :, :3].any() and not wide[:, :, 93:].any()
    tall = torch.zeros(2, 91, 70, dtype=dtype, device="cuda")
    orthogonalize(x, out=tall[:, 1:].mT)
    assert torch.equal(tall[:, 1:].mT, want) and not tall[:, 0].any()
    y = x.clone()
    assert orthogonalize(y, out=y) is y and torch.equal(y, want)


def test_scale_zeros_and_values_that_are_not_finite():
    from zeno_amd.optim import orthogonalize

    x = matrices((40, 60), torch.float32, 5).cuda()
    want = orthogonalize(x)
    for f in (2.0 ** 120, 2.0 ** 20):  # the norm's square leaves fp32's range
        assert_near(orthogonalize(x * f), reference((x * f).cpu()), 1e-4)
    assert not orthogonalize(torch.zeros_like(x)).any()
    both = torch.stack([x, x])
    both[0, 3, 4] = float("nan")
    got = orthogonalize(both)
    assert torch.isnan(got[0]).all() and torch.equal(got[1], want)  # one matrix does not reach another
    both[0, 3, 4] = float("inf")
    assert torch.equal(orthogonalize(both)[1], want)


def test_other_coefficients_and_steps():
    from zeno_amd.optim import orthogonalize

    x = matrices((50, 80), torch.float32, 6)
    for steps, coefficients in ((1, (1.5, -0.5, 0.0)), (12, (1.5, -0.5, 0.0)), (3, (3.4445, -4.7750, 2.0315))):
        assert_near(orthogonalize(x.cuda(), steps, coefficients), reference(x, steps, coefficients), 1e-4)


def test_reproducible_on_any_stream_and_in_a_graph():
    from zeno_amd.optim import orthogonalize

    x = matrices((3, 200, 260), torch.bfloat16, 7).cuda()
    want, out = orthogonalize(x), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = orthogonalize(x)
    side.synchronize()
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        orthogonalize(x, out=out)
    for seed in (8, 9, 10):
        x.copy_(matrices((3, 200, 260), torch.bfloat16, seed))
        graph.replay()
        want = orthogonalize(x)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals():
    from zeno_amd.optim import orthogonalize

    x = torch.randn(4, 5, device="cuda")
    for bad, error in [((x.double(),), TypeError), ((x[0],), ValueError), ((x[:0],), ValueError), ((x.cpu(),), ValueError), ((x, 0), ValueError),
                       ((x, 5, (3.0, 1.0, 1.0)), ValueError), ((x, 5, (1.0, 2.0)), ValueError), ((x, 5, (float("nan"), 0, 0)), ValueError),
                       ((x, 5, (1.5, -0.5, 0.0), 0.0), ValueError)]:
        with pytest.raises(error):
            orthogonalize(*bad)
    with pytest.raises(ValueError, match="out must be"):
        orthogonalize(x, out=x.half())


def test_a_matrix_written_in_place_is_noticed():
    from zeno_amd.optim import orthogonalize

    w = torch.randn(8, 8, device="cuda")
    x = torch.randn(8, 8, device="cuda", requires_grad=True)
    y = (x * w).sum()
    orthogonalize(w, out=w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(40, 250, 310), (50, 320, 250), (64, 380, 450), (130, 100, 180), (70, 128, 192)], ids=str)
def test_many_matrices_whose_sides_are_odd_numbers_of_small_tiles(shape, dtype):
    from zeno_amd.optim import orthogonalize

    x = matrices(shape, dtype, seed=7, rank=4)
    assert_near(orthogonalize(x.cuda()), reference(x), tolerance(x))
