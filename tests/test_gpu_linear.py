"""Linear attention with a decay for each head on the GPU against its definition in 64 bits: every
element type, head layout and launch shape, lengths from one token to many segments, resets, strides,
values that are not finite, and gradients.

Tolerances: outputs are rounded once (half a step of their type); before that, operands keep 24 bits and
sums are fp32. The longest chain of a value is the chunks of a walk, a chunk's tokens and the
dimensions (`work`); the sums of these inputs' terms are of random signs, so 2-norms do not cancel.
"""
import pytest
import torch

from tests.linear_reference import linear_attention as definition
from tests.policy_reference import HALF_ULP, assert_near, work_error

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ("q", "k", "v", "g", "state")


def inputs(b, t, hk, hv, dk, dv, dtype, seed, resets=0.1, slow=-4.0, fast=0.5):
    """On the CPU, rounded to the type; heads that forget slowly to fast."""
    r = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=r)

    return {"q": normal(b, t, hk, dk).to(dtype), "k": normal(b, t, hk, dk).to(dtype), "v": normal(b, t, hv, dv).to(dtype),
            "g": -torch.exp(torch.linspace(slow, fast, hv) + 0.1 * normal(hv)), "reset": torch.rand(b, t, generator=r) < resets, "state": normal(b, hv, dk, dv)}


def on_gpu(x):
    return {n: None if y is None else y.cuda() for n, y in x.items()}


def tolerance(t, dk, dv):
    return work_error(t // 32 + 32, dk, dv)


def check_train(x, scale=None, seed=0, transform=lambda n, y: y, names=NAMES, reference=None):
    from zeno_amd.memory import linear_attention as ours

    names = [n for n in names if x[n] is not None]
    ref = {n: None if y is None else (y.clone().double().requires_grad_(n in names) if y.is_floating_point() else y) for n, y in x.items()}
    dev = {n: None if y is None else transform(n, y.cuda()).detach() for n, y in x.items()}
    for n in names:
        dev[n].requires_grad_()
    o, s = definition(**ref, scale=scale)
    po, ps = ours(**dev, scale=scale)
    r = torch.Generator().manual_seed(seed + 77)
    do, ds = torch.randn(o.shape, generator=r).to(x["v"].dtype), torch.randn(s.shape, generator=r)
    want = torch.autograd.grad((o, s), [ref[n] for n in names], (do.double(), ds.double()))
    got = torch.autograd.grad((po, ps), [dev[n] for n in names], (do.cuda(), ds.cuda()))
    t, dk, dv = x["q"].shape[1], x["q"].shape[3], x["v"].shape[3]
    work, half = tolerance(t, dk, dv), HALF_ULP[x["v"].dtype]
    assert_near(po, o, half + work, "o")
    assert_near(ps, s, work, "state")
    for n, a, b in zip(names, got, want):
        assert a.dtype == x[n].dtype and a.shape == x[n].shape
        if n == "g":  # each head's by itself, as fast heads' are small
            terms = [float(c) for c in b]
            for h, (p, q) in enumerate(zip(a.double().cpu(), terms)):
                assert abs(float(p) - q) <= work * decay_size(x, h, do, ds, scale), (h, float(p), q)
        else:
            assert_near(a, b, (half if n in "qkv" else 0.0) + work, "gradient of " + n)
    return got


def decay_size(x, h, do, ds, scale):
    """The gradient of g of one head with every term taken by its size: what its rounding is relative to."""
    y = {n: None if z is None else z.double().abs() if z.is_floating_point() else z for n, z in x.items()}
    share = x["v"].shape[2] // x["q"].shape[2]
    one = {"q": y["q"][:, :, h // share:h // share + 1], "k": y["k"][:, :, h // share:h // share + 1], "v": y["v"][:, :, h:h + 1],
           "g": x["g"].double()[h:h + 1].requires_grad_(), "reset": x["reset"], "state": None if x["state"] is None else y["state"][:, h:h + 1]}
    o, s = definition(**one, scale=scale)
    total = (o * do[:, :, h:h + 1].double().abs()).sum() + (s * ds[:, h:h + 1].double().abs()).sum()
    return float(torch.autograd.grad(total, one["g"])[0])


# Batches large enough for waves of 64 columns (2048 of them), one chunk or several, whole and odd dimensions, shared heads;
# among them some whose gradients' walks, or whose values, leave such waves half idle and are given waves of 32.
MANY = [(2048, 9, 1, 1, 64, 64), (1030, 37, 1, 2, 33, 63), (700, 33, 3, 3, 64, 64), (520, 20, 2, 4, 24, 40), (2050, 3, 1, 1, 32, 48), (1030, 17, 1, 1, 20, 100),
        (700, 40, 1, 1, 64, 33), (720, 18, 1, 1, 63, 16), (1030, 20, 1, 1, 64, 80), (1000, 34, 1, 2, 32, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_many_sequences(shape, dtype):
    check_train(inputs(*shape, dtype, seed=sum(shape)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_many_sequences_with_values_that_are_not_finite(bad, dtype):
    """Waves of 64 columns: one sequence has such a value, between resets; no other row of it and no other
    sequence or head is reached."""
    from zeno_amd.memory import linear_attention as ours

    b, t, h, d = 1024, 44, 2, 64
    x = inputs(b, t, 1, h, d, d, dtype, seed=14, resets=0.05)
    x["reset"][:, 12] = x["reset"][:, 30] = True
    x["state"][7, 1] = bad  # and a state, up to its first reset
    spoilt = {n: y.clone() for n, y in x.items()}
    spoilt["v"][500, 20, 1, 40] = bad
    spoilt["k"][501, 20, 0, 3] = bad
    spoilt["q"][502, 20, 0, 63] = bad
    tol = 2 * HALF_ULP[dtype] + 2 * tolerance(t, d, d)
    results = []
    for y in (x, spoilt):
        dev = {n: z.cuda().requires_grad_(z.is_floating_point() and n != "g") for n, z in y.items()}
        o, s = ours(**dev)
        results.append([o, s, *torch.autograd.grad(o.float().square().sum() + s.square().sum(), [dev[n] for n in "qkv"])])
    clean, other = results
    apart = torch.ones(b, t, dtype=torch.bool)
    apart[500:503, 12:30] = False
    apart[7, :12] = False
    for n, p, r in zip(("o", "state", "q", "k", "v"), other, clean):
        p, r = p.cpu(), r.cpu()
        if n == "state":
            assert_near(p, r, tol, n)
            continue
        # The squares' gradient is 2 o, so that its rounding comes on top.
        assert_near(p[apart], r[apart], tol if n == "o" else 4 * tol, n)
    o, ref = other[0].cpu(), clean[0].cpu()
    assert torch.isfinite(ref[500:503]).all()
    for c in (slice(0, 40), slice(41, 64)):
        assert_near(o[500, :, 1, c], ref[500, :, 1, c], tol, "other columns")
    assert_near(o[500, :, 0], ref[500, :, 0], tol, "the other head")
    assert_near(o[502, 21:], ref[502, 21:], tol, "behind a query")
    assert not torch.isfinite(o[500, 20, 1, 40]) and not torch.isfinite(o[501, 20]).all() and not torch.isfinite(o[502, 20]).any()


def test_small_half_precision_values():
    """float16 rows below its smallest normal value: products are of the values themselves."""
    x = inputs(3, 70, 1, 2, 64, 64, torch.float16, seed=21, resets=0.05)
    for n in "qk":
        x[n] = (x[n].float() * 2.0 ** -18).half()  # 64 steps of 2^-24
    x["state"] *= 2.0 ** -18
    from zeno_amd.memory import linear_attention as ours

    # The scale brings the outputs back to normal values, of which half a step is the rounding.
    o, s = ours(**on_gpu(x), scale=2.0 ** 32)
    want, last = definition(**x, scale=2.0 ** 32)
    assert_near(o, want, HALF_ULP[torch.float16] + tolerance(70, 64, 64), "o")
    assert_near(s, last, tolerance(70, 64, 64), "state")


def test_many_heads_of_long_sequences_are_not_cut():
    """As many waves as fill the device: no segments, and many chunks to a walk."""
    check_train(inputs(128, 300, 2, 16, 8, 16, torch.bfloat16, seed=31, resets=0.01))


# (batch, length, key heads, value heads, key_dim, value_dim): every launch shape of every type,
# lengths around the chunks of 16 and 32 and of one and several segments, odd dimensions
SHAPES = [(2, 1, 1, 1, 8, 8), (3, 15, 2, 2, 16, 24), (2, 16, 1, 2, 64, 64), (2, 17, 2, 2, 32, 32), (3, 31, 1, 1, 32, 64), (2, 32, 1, 2, 64, 32), (2, 33, 2, 6, 33, 65),
          (1, 100, 1, 1, 64, 128), (2, 65, 1, 3, 128, 128), (1, 48, 2, 2, 65, 1), (1, 17, 1, 1, 1, 128), (1, 130, 1, 1, 127, 63), (1, 300, 1, 2, 64, 64),
          (2, 517, 1, 1, 40, 72), (1, 700, 2, 2, 128, 128), (40, 9, 2, 4, 24, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sequences_and_gradients(shape, dtype):
    check_train(inputs(*shape, dtype, seed=sum(shape), resets=0.1 if shape[1] < 200 else 0.003))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 70, 2, 4, 40, 72), (1, 400, 1, 2, 64, 64)], ids=str)
def test_other_scale_no_state_no_reset_no_decay_gradient(shape, dtype):
    x = inputs(*shape, dtype, seed=5)
    x["state"] = x["reset"] = None
    check_train(x, scale=0.37)
    check_train(x, names=("q", "k", "v"))
    check_train(inputs(*shape, dtype, seed=6, resets=0.02), names=("q", "k", "v", "state"))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(5, 1, 1, 8, 8), (3, 2, 6, 64, 64), (2, 1, 4, 128, 128), (7, 1, 1, 70, 37), (2, 3, 3, 32, 121), (1, 1, 2, 17, 1)], ids=str)
def test_step(shape, dtype):
    from zeno_amd.memory import linear_attention_step

    b, hk, hv, dk, dv = shape
    x = inputs(b, 3, hk, hv, dk, dv, dtype, seed=sum(shape), resets=0.3)
    o, s = definition(**x)
    d = on_gpu(x)
    state = d.pop("state")
    got = torch.stack([linear_attention_step(*(d[n][:, t] for n in "qkv"), d["g"], state, d["reset"][:, t]) for t in range(3)], 1)
    assert_near(got, o, HALF_ULP[dtype] + work_error(3, dk), "o")
    assert_near(state, s, work_error(3, dk), "state")


def test_steps_agree_with_the_sequence():
    """A rollout acted token by token and then trained on as a whole: the same outputs."""
    from zeno_amd.memory import linear_attention as ours, linear_attention_step

    x = on_gpu(inputs(64, 50, 2, 4, 64, 64, torch.float32, seed=9, resets=0.05))
    state = x["state"].clone()
    o, last = ours(**x)
    steps = torch.stack([linear_attention_step(*(x[n][:, t] for n in "qkv"), x["g"], state, x["reset"][:, t]) for t in range(50)], 1)
    assert_near(steps, o, 2 * work_error(50, 64), "o")
    assert_near(state, last, 2 * work_error(50, 64), "state")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_segments_agree_with_parts(dtype):
    """One long sequence, walked in segments, against the same handed on from part to part."""
    from zeno_amd.memory import linear_attention as ours

    x = on_gpu(inputs(1, 2500, 1, 2, 64, 64, dtype, seed=2, resets=0.001, slow=-5.0))
    o, last = ours(**x)
    state, outs = x["state"], []
    for t in range(0, 2500, 100):
        part, state = ours(*(x[n][:, t:t + 100] for n in "qkv"), x["g"], x["reset"][:, t:t + 100], state)
        outs.append(part)
    tol = 2 * work_error(80, 64, 64)
    assert_near(torch.cat(outs, 1), o, 2 * HALF_ULP[dtype] + tol, "o")
    assert_near(state, last, tol, "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_time_major_views_and_odd_addresses(dtype):
    """Views of one projection, recorded time-major; rows at any address; broadcast inputs; gradients
    keep the inputs' order."""
    from zeno_amd.memory import linear_attention as ours

    x = inputs(3, 45, 2, 2, 24, 40, dtype, seed=3)
    check_train(x, transform=lambda n, y: y if n in ("g", "state") else y.transpose(0, 1).contiguous().transpose(0, 1))
    d = on_gpu(x)
    want = ours(**d)
    fused = torch.cat([d[n].flatten(2) for n in "qkv"], -1)
    q, k, v = (y.unflatten(-1, (2, -1)) for y in fused.split([48, 48, 80], -1))
    got = ours(q, k, v, d["g"], d["reset"], d["state"])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.zeros(3, 45, 2, 24 + 24 + 40 + 5, dtype=dtype, device="cuda")  # heads at odd addresses
    q, k, v = wide[..., 1:25], wide[..., 26:50], wide[..., 52:92]
    for n, y in (("q", q), ("k", k), ("v", v)):
        y.copy_(d[n])
    got = ours(q, k, v, d["g"], d["reset"], d["state"])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = {n: d[n][:1] for n in ("q", "k", "v", "reset", "state")}
    got = ours(*(one[n].expand(4, *one[n].shape[1:]) for n in "qkv"), d["g"], one["reset"].expand(4, 45), one["state"].expand(4, 2, 24, 40))
    assert all(torch.equal(a[i], b[0]) for a, b in zip(got, want) for i in range(4))
    leaf = d["v"][:1].detach().requires_grad_()
    o, _ = ours(d["q"], d["k"], leaf.expand(3, 45, 2, 40), d["g"], d["reset"], d["state"])
    (grad,) = torch.autograd.grad(o.float().sum(), leaf)
    assert grad.shape == leaf.shape and torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("g", [0.0, -1e-4, -8.0, -16.0, -40.0, -150.0, float("-inf"), 0.03])
def test_decays(g, dtype):
    """Heads that keep everything, forget fast, at once, or grow; gradients of fast decays keep their digits."""
    for t in (40, 260):
        x = inputs(2, t, 1, 2, 32, 48, dtype, seed=11, resets=0.02)
        x["g"] = torch.tensor([g, -0.5])
        check_train(x, names=NAMES if g > -80 else ("q", "k", "v", "state"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_heads_that_grow_fast(dtype):
    """exp(3 * 32) passes fp32's range, exp(3 * 9) does not: nothing is multiplied by what 32 tokens would make of it."""
    for t in (3, 9, 18):
        x = inputs(2, t, 1, 2, 32, 48, dtype, seed=13, resets=0.0)
        x["g"] = torch.tensor([3.0, -0.5])
        check_train(x)


def test_decay_gradient_of_heads_that_forget_at_once():
    from zeno_amd.memory import linear_attention as ours

    x = on_gpu(inputs(2, 40, 1, 2, 16, 16, torch.float32, seed=1))
    g = torch.tensor([float("-inf"), -200.0], device="cuda").requires_grad_()
    o, _ = ours(x["q"], x["k"], x["v"], g, x["reset"], x["state"])
    assert torch.equal(torch.autograd.grad(o.sum(), g)[0], torch.zeros_like(g))


@pytest.mark.parametrize("resets", ["first", "all", "last", "chunk ends", "uint8"])
def test_resets(resets):
    x = inputs(3, 100, 1, 2, 40, 64, torch.float32, seed=8, resets=0.0)
    flags = x["reset"]
    if resets == "first":
        flags[:, 0] = True
    elif resets == "all":
        flags[:] = True
    elif resets == "last":
        flags[:, -1] = True
    elif resets == "chunk ends":
        flags[:, [15, 16, 31, 32, 63, 64]] = True
    else:
        flags[:, [3, 50]] = True
        x["reset"] = flags.to(torch.uint8) * 255
    check_train(x)
    x = inputs(1, 400, 1, 1, 64, 64, torch.float32, seed=8, resets=0.0)  # the same across segments
    x["reset"][:, [0, 127, 128, 255, 256, 399]] = True
    check_train(x)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite(bad, dtype):
    """They reach no output before their token, none behind a reset, and of the values no other column."""
    from zeno_amd.memory import linear_attention as ours

    for t, length in ((37, 90), (5, 20), (140, 500)):
        x = inputs(2, length, 1, 1, 40, 64, dtype, seed=4, resets=0.0)
        x["reset"][:, t + 9] = True
        clean = ours(**on_gpu(x))
        for n in "qkv":
            y = {m: z.clone() for m, z in x.items()}
            y[n][0, t, 0, 7] = bad
            o, last = ours(**on_gpu(y))
            apart = torch.ones(2, length, dtype=torch.bool)
            apart[0, t:t + 9] = False
            if n == "q":
                apart[0, t + 1:] = True
            tol = HALF_ULP[dtype] * 2 + tolerance(length, 40, 64)
            assert_near(o.cpu()[apart], clean[0].cpu()[apart], tol, n)
            assert_near(last, clean[1], tol, "state")
            assert not torch.isfinite(o[0, t]).all()
            if n == "v":
                others = [c for c in range(64) if c != 7]
                assert_near(o[0][..., others], clean[0][0][..., others], tol, "other columns")
        # gradients: of a NaN in the gradient of o, up to its token and not beyond the reset before it
        x["reset"][:, t - 4] = True
        d = {m: z.cuda().requires_grad_(z.is_floating_point()) for m, z in x.items()}
        grads = []
        for value in (0.5, bad):
            d_o = torch.ones_like(clean[0])
            d_o[0, t, 0, 7] = value
            o, _ = ours(**d)
            grads.append(torch.autograd.grad(o, [d[n] for n in "qkv"], d_o))
        for n, a, b in zip("qkv", *grads):
            apart = torch.ones(2, length, dtype=torch.bool)
            apart[0, t - 4:t + 1] = False
            assert_near(b.cpu()[apart], a.cpu()[apart], HALF_ULP[dtype] * 2 + tolerance(length, 40, 64), "gradient of " + n)


def test_a_state_that_is_not_finite_passes_no_reset():
    from zeno_amd.memory import linear_attention as ours, linear_attention_step

    x = on_gpu(inputs(1, 70, 1, 1, 32, 32, torch.float32, seed=4, resets=0.0))
    for t in (0, 20, 40):
        x["reset"][:] = False
        x["reset"][:, t] = True
        want, keep = ours(**x), x["state"].clone()
        for bad in (float("nan"), float("inf")):
            x["state"] = torch.full_like(keep, bad)
            o, last = ours(**x)
            # Token by token where the reset is: the same terms in another order, each sum within the tolerance.
            assert_near(o[:, t:], want[0][:, t:], 2 * tolerance(70, 32, 32), "o")
            assert_near(last, want[1], 2 * tolerance(70, 32, 32), "state")
            state = torch.full_like(keep, bad)
            linear_attention_step(*(x[n][:, 0] for n in "qkv"), x["g"], state, torch.ones(1, dtype=torch.bool, device="cuda"))
            assert torch.isfinite(state).all()
        x["state"] = keep


def test_gradients_against_differences():
    """Central differences of the definition in 64 bits, one direction an input at a time: off by h^2 and
    the kernel's own roundings."""
    from zeno_amd.memory import linear_attention as ours

    x = inputs(2, 50, 1, 2, 12, 20, torch.float32, seed=12, resets=0.05)
    dev = {n: y.cuda().requires_grad_(n in NAMES) for n, y in x.items()}
    r = torch.Generator().manual_seed(5)
    o, s = ours(**dev)
    c = [torch.randn(o.shape, generator=r), torch.randn(s.shape, generator=r)]
    grads = torch.autograd.grad((o, s), [dev[n] for n in NAMES], [z.cuda() for z in c])
    h = 1e-4
    for n, g in zip(NAMES, grads):
        d = torch.randn(x[n].shape, generator=r, dtype=torch.float64)

        def value(step):
            y = {m: z.double() if z.is_floating_point() else z for m, z in x.items()}
            y[n] = y[n] + step * d
            o, s = definition(**y)
            return float((o * c[0]).sum() + (s * c[1]).sum())

        slope, size = (value(h) - value(-h)) / (2 * h), float(g.double().norm().cpu() * d.norm())
        assert abs(float((g.double().cpu() * d).sum()) - slope) <= size * (1e-5 + tolerance(50, 12, 20)), n


def test_only_one_gradient_comes_in():
    from zeno_amd.memory import linear_attention as ours

    for t in (40, 300):
        x = inputs(1, t, 1, 2, 32, 32, torch.float32, seed=3, resets=0.02)
        for which in (0, 1):
            ref = {n: y.double().requires_grad_() if y.is_floating_point() else y for n, y in x.items()}
            dev = {n: y.cuda().requires_grad_(y.is_floating_point()) for n, y in x.items()}
            a, b = definition(**ref)[which], ours(**dev)[which]
            names = NAMES if which == 0 else ("k", "v", "g", "state")
            want = torch.autograd.grad((a * a).sum(), [ref[n] for n in names])
            got = torch.autograd.grad((b * b).sum(), [dev[n] for n in names])
            for n, p, q in zip(names, got, want):
                assert_near(p, q, 4 * tolerance(t, 32, 32), n)


def test_runs_are_bitwise_alike():
    x = inputs(3, 333, 2, 4, 24, 48, torch.float32, seed=1, resets=0.01)
    a, b = check_train(x), check_train(x)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_streams_and_graph():
    """On a stream of its own, and captured with its gradients into a graph that is replayed with other
    inputs, eager work between the replays."""
    from zeno_amd.memory import linear_attention as ours

    for t in (40, 600):
        x = on_gpu(inputs(2, t, 1, 2, 64, 64, torch.bfloat16, seed=3, resets=0.02))
        d_o, d_s = torch.randn(2, t, 2, 64, device="cuda").bfloat16(), torch.randn(2, 2, 64, 64, device="cuda")

        def run(z):
            leaves = {n: y.detach().requires_grad_(n in NAMES) for n, y in z.items()}
            o, s = ours(**leaves)
            return [o.detach(), s.detach(), *torch.autograd.grad((o, s), [leaves[n] for n in NAMES], (d_o, d_s))]

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
            for n in NAMES:
                held[n].copy_(x[n] * (1 + i / 4))
            eager = run(held)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_refusals():
    from zeno_amd.memory import linear_attention as ours, linear_attention_step

    x = on_gpu(inputs(2, 6, 1, 2, 16, 24, torch.float32, seed=1))
    for change, kind in ((dict(g=x["g"].double()), TypeError), (dict(g=x["g"][:1]), ValueError), (dict(g=x["g"][None]), ValueError), (dict(q=x["q"].half()), TypeError),
                         (dict(q=x["q"].double(), k=x["k"].double(), v=x["v"].double()), TypeError), (dict(k=x["k"][:1]), ValueError), (dict(v=x["v"][:, :5]), ValueError),
                         (dict(g=x["g"].cpu()), ValueError), (dict(state=x["state"].half()), TypeError), (dict(state=x["state"][:1]), ValueError),
                         (dict(reset=x["reset"].float()), TypeError), (dict(reset=x["reset"][:, :5]), ValueError), (dict(scale=float("inf")), ValueError),
                         (dict(q=x["q"].cpu()), ValueError), (dict(v=x["v"].repeat(1, 1, 1, 6)), ValueError), (dict(v=x["v"][..., :0]), ValueError)):
        with pytest.raises(kind):
            ours(**{**x, **change})
    with pytest.raises(ValueError):  # three value heads on two key heads
        ours(x["q"].repeat(1, 1, 2, 1), x["k"].repeat(1, 1, 2, 1), x["v"][:, :, :1].repeat(1, 1, 3, 1), x["g"][:1].repeat(3))
    token = [x[n][:, 0] for n in "qkv"]
    for state, out in ((x["state"].transpose(2, 3).contiguous().transpose(2, 3), None), (x["state"].clone().requires_grad_(), None),
                       (x["state"], token[2].half()), (x["state"], x["state"][:, :, 0]), (x["state"], token[2][:1].expand(2, 2, 24)), (x["state"], token[2][..., ::2])):
        with pytest.raises(ValueError):
            linear_attention_step(*token, x["g"], state, out=out)
    s = x["state"].clone()
    v = token[2].clone()
    want = linear_attention_step(*token, x["g"], x["state"])
    assert linear_attention_step(token[0], token[1], v, x["g"], s, out=v) is v and torch.equal(v, want)


def test_places_behind_2_31_elements():
    """One sequence whose values, and wide rows whose strides, go beyond 2^31 elements: the last tokens agree with a short call's."""
    from zeno_amd.memory import linear_attention as ours

    t, part = (1 << 22) + 70, 200
    r = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.empty(1, t, 2, 8 + 8 + 256, dtype=torch.float16, device="cuda")  # 2^31 elements and more; the heads are slices of it
    q, k, v = wide[..., :8], wide[..., 8:16], wide[..., 16:48]
    for x in (q, k, v):
        x.copy_(torch.randn(x.shape, generator=r, device="cuda", dtype=torch.float16))
    assert wide.numel() > 1 << 31
    g = torch.tensor([-1.0, -0.7], device="cuda")
    reset = torch.zeros(1, t, dtype=torch.bool, device="cuda")
    reset[0, t - part] = True
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o, last = ours(*leaves, g, reset)
    tail = [x[:, t - part:].clone().requires_grad_() for x in (q, k, v)]
    want, end = ours(*tail, g)
    tol = 2 * HALF_ULP[torch.float16] + 2 * tolerance(part, 8, 32)
    assert_near(o[:, t - part:], want, tol, "o")
    assert_near(last, end, 2 * tolerance(part, 8, 32), "state")
    d_o = torch.zeros_like(o)
    d_o[:, t - part:] = torch.randn(want.shape, generator=r, device="cuda", dtype=torch.float16)
    got = torch.autograd.grad(o, leaves, d_o)
    ref = torch.autograd.grad(want, tail, d_o[:, t - part:].contiguous())
    for n, a, b in zip("qkv", got, ref):
        assert a.abs().sum(dtype=torch.float64).isfinite()
        assert_near(a[:, t - part:], b, tol, "gradient of " + n)
        assert not a[:, :t - part].any(), n
