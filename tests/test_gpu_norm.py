"""Layer norm on the GPU against its definition in 64 bits: every element type, launch shape and kind
of weights, rows of any stride, rows off zero, gradients, streams and graphs.

Tolerances: y is rounded once (half a step of its type); before that every value passes sums of at
most 16 terms in a lane, 64 lanes and 16 waves (chains of 16 + 6 + 16 additions) and about ten further
roundings, `ROW` in all. Sums over rows add chains of rows / 512 (in a lane), the workgroup's rows and
the workgroups / 32 of a slice and 32 slices.
"""
import pytest
import torch

from tests.norm_reference import layer_norm as definition
from tests.policy_reference import HALF_ULP, assert_near, work_error

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ROW = work_error(48)


def column_sum(rows):
    return ROW + work_error(rows // 512 + 16 + 32 + 32)


def inputs(shape, dtype, weights, seed, residual=False, offset=0.5):
    r = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=r)

    n = shape[-1]
    x = {"x": (normal(*shape) + offset * normal(n)).to(dtype), "weight": (1.0 + 0.3 * normal(n)).to(weights), "bias": (0.3 * normal(n)).to(weights)}
    if residual:
        x["residual"] = (2.0 * normal(*shape)).to(dtype)
    return x


def check(x, eps=1e-5, seed=0, transform=lambda n, y: y):
    from zeno_amd.norm import layer_norm

    ref = {n: y.double().requires_grad_() for n, y in x.items()}
    dtype = x["x"].dtype
    if "residual" in x:  # the definition rounds sums to the operator's type
        exact = ref["x"] + ref["residual"]
        total = exact + (exact.detach().to(dtype).double() - exact.detach())
        want = (definition(total, ref.get("weight"), ref.get("bias"), eps=eps), total)
    else:
        want = (definition(**ref, eps=eps),)
    dev = {n: transform(n, y.cuda()).detach().requires_grad_() for n, y in x.items()}
    got = layer_norm(dev["x"], dev.get("weight"), dev.get("bias"), residual=dev.get("residual"), eps=eps)
    got = got if "residual" in x else (got,)
    r = torch.Generator().manual_seed(seed + 77)
    d = [torch.randn(y.shape, generator=r).to(dtype) for y in want]
    rows, half = x["x"].numel() // x["x"].shape[-1], HALF_ULP[dtype]
    assert got[0].dtype == dtype and got[0].shape == x["x"].shape
    assert_near(got[0], want[0], half + ROW, "y")
    if "residual" in x:
        assert torch.equal(got[1].cpu(), want[1].to(dtype))
    names = list(x)
    want = torch.autograd.grad(want, [ref[n] for n in names], [y.double() for y in d])
    got = torch.autograd.grad(got, [dev[n] for n in names], [y.cuda() for y in d])
    for n, a, b in zip(names, got, want):
        assert a.dtype == x[n].dtype and a.shape == x[n].shape
        if n in ("weight", "bias"):
            assert_near(a, b, HALF_ULP[a.dtype] + column_sum(rows), "gradient of " + n)
        else:
            assert_near(a, b, half + 2 * ROW, "gradient of " + n)
    return got


# One size for every launch shape, exact and not: lanes of 8 to 1024, one and two vectors.
SHAPES = [(1, 1), (3, 7), (1, 8), (33, 64), (5, 63), (2, 3, 5, 128), (70, 65), (9, 256), (7, 129), (5, 512), (2, 511), (3, 1024), (4, 1000),
          (2, 2048), (3, 1025), (2, 4096), (3, 2049), (2, 8192), (2, 4097), (2, 16384), (3, 16381)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows_and_gradients(shape, dtype):
    check(inputs(shape, dtype, torch.float32, seed=sum(shape)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 37, 64), (3, 100), (5, 1000), (2, 8191)], ids=str)
def test_residual_sums(shape, dtype):
    x = inputs(shape, dtype, dtype, seed=sum(shape), residual=True)
    dx, _, _, d_residual = check(x)
    assert torch.equal(dx, d_residual)


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 5000, 40001])
def test_numbers_of_rows(rows):
    """More rows than the workgroups take at a time, and an odd rest of them."""
    check(inputs((rows, 40), torch.float32, torch.float32, seed=rows))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_without_weight_or_bias(dtype):
    for drop in (("weight",), ("bias",), ("weight", "bias")):
        x = inputs((6, 50), dtype, torch.float32, seed=2)
        check({n: y for n, y in x.items() if n not in drop})


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n", [48, 250, 1500])
def test_strides(n, dtype):
    """Parts of wider rows at odd addresses, time-major rows, broadcast rows, more dimensions than three,
    features that are not contiguous: the same bits as of copies."""
    from zeno_amd.norm import layer_norm

    x = inputs((3, 4, 5, n), dtype, torch.float32, seed=n)

    def slices(name, y):
        if y.dim() == 1:
            return y
        wide = torch.zeros(*y.shape[:-1], n + 7, dtype=dtype, device="cuda")
        wide[..., 3:3 + n] = y
        return wide[..., 3:3 + n]

    check(x, transform=slices)
    check(x, transform=lambda name, y: y if y.dim() == 1 else y.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3))
    check(x, transform=lambda name, y: y if y.dim() == 1 else y.transpose(1, 3).contiguous().transpose(1, 3))
    d = {name: y.cuda() for name, y in x.items()}
    want = layer_norm(**d)
    assert torch.equal(layer_norm(d["x"].view(3, 2, 2, 5, 1, n), d["weight"], d["bias"]).view_as(want), want)
    one = d["x"][:1, :, 2:3]
    assert torch.equal(layer_norm(one.expand(6, 4, 5, n), d["weight"], d["bias"]), layer_norm(one, d["weight"], d["bias"]).expand(6, 4, 5, n))
    y = layer_norm(d["x"].permute(2, 0, 1, 3), d["weight"], d["bias"])
    assert torch.equal(y, want.permute(2, 0, 1, 3))


def test_broadcast_inputs_and_gradients():
    """Inputs and gradients that repeat memory: each place gets its own gradient, summed by autograd."""
    from zeno_amd.norm import layer_norm

    x = inputs((1, 24), torch.float32, torch.float32, seed=4)
    ref = {n: y.double().requires_grad_() for n, y in x.items()}
    dev = {n: y.cuda().requires_grad_() for n, y in x.items()}
    want = definition(ref["x"].expand(50, 24), ref["weight"], ref["bias"])
    got = layer_norm(dev["x"].expand(50, 24), dev["weight"], dev["bias"])
    c = torch.randn(24, generator=torch.Generator().manual_seed(1))
    a = torch.autograd.grad((got * c.cuda()).sum(), list(dev.values()))
    b = torch.autograd.grad((want * c.double()).sum(), list(ref.values()))
    for p, q, n in zip(a, b, dev):
        assert_near(p, q, 2 * column_sum(50), n)
    got = layer_norm(dev["x"].expand(50, 24), dev["weight"], dev["bias"])
    (a,) = torch.autograd.grad(got.sum(), dev["bias"])
    assert torch.equal(a, torch.full_like(a, 50.0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_far_off_zero(dtype):
    """A row 1000 of its own sizes off zero (in fp32: 10000) keeps its digits."""
    r = torch.Generator().manual_seed(3)
    far = 1e4 if dtype == torch.float32 else 4.0 / HALF_ULP[dtype] ** 0.5
    x = {"x": (far + torch.randn(20, 300, generator=r)).to(dtype), "weight": torch.ones(300), "bias": torch.zeros(300)}
    check(x)


def test_constant_and_tiny_rows():
    """A row without variance gives the bias; rows whose variance is below eps, and eps 0."""
    from zeno_amd.norm import layer_norm

    x = torch.full((3, 65), 3.7, device="cuda")
    bias = torch.randn(65, device="cuda")
    y = layer_norm(x, None, bias)
    assert float((y - bias).abs().max()) <= 3.7 * 2 ** -24 / 1e-5 ** 0.5  # the mean's last digit over sqrt(eps)
    check(inputs((4, 33), torch.float32, torch.float32, seed=8), eps=3.0)
    check(inputs((4, 33), torch.float32, torch.float32, seed=8), eps=0.0)


def test_values_that_are_not_finite_stay_in_their_row():
    from zeno_amd.norm import layer_norm

    for n in (64, 100, 5000):
        x = torch.randn(9, n, device="cuda")
        want = layer_norm(x)
        for bad in (float("nan"), float("inf"), -float("inf")):
            z = x.clone()
            z[4, n // 2] = bad
            y = layer_norm(z)
            assert torch.isnan(y[4]).all()
            y[4] = want[4]
            assert torch.equal(y, want)


def test_gradients_against_differences():
    """Central differences of the definition in 64 bits, one direction an input at a time: off by the
    third derivative, h^2, and the kernel's own roundings."""
    from zeno_amd.norm import layer_norm

    x = inputs((6, 37), torch.float32, torch.float32, seed=12, residual=True)
    dev = {n: y.cuda().requires_grad_() for n, y in x.items()}
    r = torch.Generator().manual_seed(5)
    c = [torch.randn(6, 37, generator=r) for _ in range(2)]
    y = layer_norm(dev["x"], dev["weight"], dev["bias"], residual=dev["residual"])
    grads = torch.autograd.grad(y, list(dev.values()), [z.cuda() for z in c])

    def value(**z):  # without the rounding of the sums, which no difference sees
        s = z["x"] + z["residual"]
        return float((definition(s, z["weight"], z["bias"]) * c[0]).sum() + (s * c[1]).sum())

    h = 1e-4
    for n, g in zip(dev, grads):
        d = torch.randn(x[n].shape, generator=r, dtype=torch.float64)
        ref = {m: z.double() for m, z in x.items()}
        up, down = (value(**{**ref, n: ref[n] + s * h * d}) for s in (1, -1))
        slope, size = (up - down) / (2 * h), float(g.double().norm().cpu() * d.norm())
        assert abs(float((g.double().cpu() * d).sum()) - slope) <= size * (1e-6 + ROW + 2.0 ** -24 * 4), n


def test_only_the_gradients_that_are_wanted():
    from zeno_amd.norm import layer_norm

    x = {n: y.cuda() for n, y in inputs((7, 80), torch.float32, torch.float32, seed=6, residual=True).items()}
    leaves = {n: y.clone().requires_grad_() for n, y in x.items()}
    d = [torch.randn(7, 80, device="cuda") for _ in range(2)]

    def grads(names, which=(0, 1)):
        z = {n: leaves[n] if n in names else x[n] for n in x}
        y = layer_norm(z["x"], z["weight"], z["bias"], residual=z["residual"])
        return torch.autograd.grad([y[i] for i in which], [z[n] for n in names], [d[i] for i in which])

    all_of = dict(zip(x, grads(list(x))))
    for n in x:
        assert torch.equal(grads([n])[0], all_of[n])
    assert torch.equal(grads(["weight", "bias"])[1], all_of["bias"])
    # One output alone: of the sum's gradient nothing is normalised.
    assert torch.equal(grads(["x"], (1,))[0], d[1])
    a, b = grads(["x"], (0,))[0], all_of["x"]
    assert_near(a + d[1], b, 2.0 ** -22, "x")


def test_runs_are_bitwise_alike():
    x = inputs((3001, 129), torch.bfloat16, torch.float32, seed=1)
    a, b = check(x), check(x)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_streams_and_graph():
    """On a stream of its own, and captured with its gradients into a graph that is replayed with other
    inputs, eager work between the replays."""
    from zeno_amd.norm import layer_norm

    x = {n: y.cuda() for n, y in inputs((300, 200), torch.float32, torch.float32, seed=3, residual=True).items()}
    d = torch.randn(2, 300, 200, device="cuda")

    def run(z):
        leaves = [z[n].detach().requires_grad_() for n in ("x", "weight", "bias", "residual")]
        y = layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3])
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, list(d)))

    want = run(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, held = torch.cuda.CUDAGraph(), {n: y.clone() for n, y in x.items()}
    with torch.cuda.stream(side):
        run(held)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = run(held)
    for i in range(4):
        for n in held:
            held[n].copy_(x[n] * (1 + i))
        eager = run(held)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_refusals():
    from zeno_amd.norm import layer_norm

    x = torch.zeros(4, 8, device="cuda")
    for bad, kind in ((dict(x=x.double()), TypeError), (dict(x=x.cpu()), ValueError), (dict(x=x[:0]), ValueError), (dict(x=x[:, :0]), ValueError),
                      (dict(x=x[0, 0]), ValueError), (dict(weight=x[0, :7]), ValueError), (dict(weight=x[0].half()), TypeError),
                      (dict(bias=x), ValueError), (dict(bias=x[0].cpu()), ValueError), (dict(weight=x[0], bias=x[0].double()), TypeError),
                      (dict(residual=x[:2]), ValueError), (dict(residual=x.half()), ValueError), (dict(residual=x.cpu()), ValueError),
                      (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError), (dict(x=torch.zeros(2, 16385, device="cuda")), ValueError)):
        with pytest.raises(kind):
            layer_norm(**{"x": x, **bad})
    h = x.half()
    with pytest.raises(TypeError):  # two types
        layer_norm(h, h[0], x[0])


def test_places_behind_2_31_elements():
    """Rows of a wide tensor beyond 2^31 elements: the last ones agree with a short call's."""
    from zeno_amd.norm import layer_norm

    wide = torch.empty((1 << 20) + 3, 2112, dtype=torch.float16, device="cuda")
    x = wide[:, 5:37]
    x.copy_(torch.randn(x.shape, device="cuda"))
    assert x.stride(0) * (len(x) - 1) > 1 << 31
    leaf = x.detach().requires_grad_()
    y = layer_norm(leaf)
    assert torch.equal(y[-70:], layer_norm(x[-70:].clone()))
    d = torch.randn_like(y)
    tail = x[-70:].clone().requires_grad_()
    (got,), (want,) = torch.autograd.grad(y, leaf, d), torch.autograd.grad(layer_norm(tail), tail, d[-70:].contiguous())
    assert torch.equal(got[-70:], want)
