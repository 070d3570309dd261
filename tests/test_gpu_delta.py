"""The gated delta rule on the GPU against its definition in 64 bits: every element type, head
layout and launch shape, lengths from one token, resets, strides, and gradients."""
import pytest
import torch

from tests.policy_reference import HALF_ULP, assert_near, gated_delta, work_error

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ("q", "k", "v", "g", "beta", "state")


def inputs(b, t, hk, hv, dk, dv, dtype, seed, resets=0.1, normalize=True):
    """On the CPU, rounded to the type; moderate keys where they are not normalised."""
    r = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=r)

    f = 1.0 if normalize else dk ** -0.5
    x = {"q": (normal(b, t, hk, dk) * f).to(dtype), "k": (normal(b, t, hk, dk) * f).to(dtype), "v": normal(b, t, hv, dv).to(dtype),
         "g": -torch.nn.functional.softplus(normal(b, t, hv)) * torch.linspace(0.01, 1.0, hv), "beta": torch.sigmoid(normal(b, t, hv)),
         "reset": torch.rand(b, t, generator=r) < resets, "state": 0.3 * normal(b, hv, dk, dv)}
    return x


def on_gpu(x):
    return {n: None if y is None else y.cuda() for n, y in x.items()}


def check_train(x, normalize, scale=None, seed=0, transform=lambda n, y: y):
    from zeno_amd.memory import gated_delta as ours

    x = dict(x)
    ref = {n: None if y is None else (y.clone().double().requires_grad_() if y.is_floating_point() else y) for n, y in x.items()}
    dev = {n: None if y is None else transform(n, y.cuda()).detach() for n, y in x.items()}
    for n in NAMES:
        if dev[n] is not None:
            dev[n].requires_grad_()
    o, s = gated_delta(**ref, scale=scale, normalize=normalize)
    po, ps = ours(**dev, scale=scale, normalize=normalize)
    r = torch.Generator().manual_seed(seed + 77)
    do, ds = torch.randn(o.shape, generator=r).to(x["v"].dtype), torch.randn(s.shape, generator=r)
    names = [n for n in NAMES if x[n] is not None]
    want = torch.autograd.grad((o, s), [ref[n] for n in names], (do.double(), ds.double()))
    got = torch.autograd.grad((po, ps), [dev[n] for n in names], (do.cuda(), ds.cuda()))
    t, dk, dv = x["q"].shape[1], x["q"].shape[3], x["v"].shape[3]
    work = work_error(t, dk, dv, 64)
    half = HALF_ULP[x["v"].dtype]
    assert_near(po, o, half + work, "o")
    assert_near(ps, s, work, "state")
    for n, a, b in zip(names, got, want):
        assert a.dtype == x[n].dtype
        assert_near(a, b, (half if n in "qkv" else 0.0) + work * (4 if n == "g" else 1), "gradient of " + n)


# (batch, length, key heads, value heads, key_dim, value_dim): every launch shape of every type,
# lengths around the chunks of 16 and 32, odd dimensions
SHAPES = [(2, 1, 1, 1, 8, 8), (3, 31, 2, 2, 16, 24), (2, 32, 1, 2, 64, 64), (2, 33, 2, 6, 33, 65), (1, 100, 1, 1, 64, 128),
          (2, 65, 1, 3, 128, 128), (1, 48, 2, 2, 65, 1), (1, 17, 1, 1, 1, 128), (1, 130, 1, 1, 127, 63)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sequences_and_gradients(shape, dtype):
    check_train(inputs(*shape, dtype, seed=sum(shape)), normalize=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_raw_keys_other_scale_no_state_no_reset(dtype):
    x = inputs(2, 70, 2, 4, 40, 72, dtype, seed=5, normalize=False)
    x["state"] = x["reset"] = None
    check_train(x, normalize=False, scale=0.37)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(5, 1, 1, 8, 8), (3, 2, 6, 64, 64), (2, 1, 4, 128, 128), (7, 1, 1, 70, 37), (2, 3, 3, 32, 121), (1, 1, 2, 17, 1)], ids=str)
def test_step(shape, dtype):
    from zeno_amd.memory import gated_delta_step

    b, hk, hv, dk, dv = shape
    x = inputs(b, 3, hk, hv, dk, dv, dtype, seed=sum(shape), resets=0.3)
    o, s = gated_delta(**x, normalize=True)
    d = on_gpu(x)
    state = d.pop("state")
    got = torch.stack([gated_delta_step(*(d[n][:, t] for n in NAMES[:5]), state, d["reset"][:, t], normalize=True) for t in range(3)], 1)
    assert_near(got, o, HALF_ULP[dtype] + work_error(3, dk), "o")
    assert_near(state, s, work_error(3, dk), "state")


def test_steps_agree_with_the_sequence():
    """A rollout acted token by token and then trained on as a whole: the same outputs."""
    from zeno_amd.memory import gated_delta as ours, gated_delta_step

    x = on_gpu(inputs(64, 50, 2, 4, 64, 64, torch.float32, seed=9, resets=0.05))
    state = x["state"].clone()
    o, last = ours(**x, normalize=True)
    steps = torch.stack([gated_delta_step(*(x[n][:, t] for n in NAMES[:5]), state, x["reset"][:, t], normalize=True) for t in range(50)], 1)
    assert_near(steps, o, 2 * work_error(50, 64, 64), "o")
    assert_near(state, last, 2 * work_error(50, 64, 64), "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_time_major_and_views(dtype):
    """Views of one projection, recorded time-major; gradients keep the inputs' order."""
    from zeno_amd.memory import gated_delta as ours

    x = inputs(3, 45, 2, 2, 24, 40, dtype, seed=3)

    def time_major(n, y):
        if n in ("state",):
            return y
        return y.transpose(0, 1).contiguous().transpose(0, 1)

    check_train(x, normalize=True, transform=time_major)
    d = on_gpu(x)
    fused = torch.cat([d[n].flatten(2) for n in "qkv"], -1)
    q, k, v = (y.unflatten(-1, (2, -1)) for y in fused.split([48, 48, 80], -1))
    a = ours(q, k, v, d["g"], d["beta"], d["reset"], d["state"], normalize=True)
    b = ours(**d, normalize=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # a last dimension that is not contiguous, and broadcast scalars
    a = ours(d["q"].mT.contiguous().mT, d["k"], d["v"], d["g"][:, :1].expand(3, 45, 2), d["beta"], d["reset"][:1].expand(3, 45), d["state"])
    b = ours(d["q"], d["k"], d["v"], d["g"][:, :1].expand(3, 45, 2).contiguous(), d["beta"], d["reset"][:1].expand(3, 45).contiguous(), d["state"])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("shape", [(2, 70, 1, 2, 24, 40), (1, 64, 1, 1, 128, 128)], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
def test_nothing_passes_a_reset(shape, bad):
    """NaN, infinities and huge values before a reset, in the state and in every operand, leave
    what follows as it is, forward and backward; resets by flag and by g = -inf."""
    from zeno_amd.memory import gated_delta as ours, gated_delta_step

    x = inputs(*shape, torch.float32, seed=11, resets=0.0)
    cut = 37
    x["reset"][:, cut] = True
    clean = on_gpu(x)
    dirty = on_gpu(x)
    for n in ("q", "k", "v", "beta"):
        dirty[n][:, cut - 3] = bad
    dirty["g"][:, cut - 5] = float("nan")
    dirty["state"][:] = bad
    flagged = dict(dirty, reset=None, g=dirty["g"].clone())
    flagged["g"][:, cut] = -float("inf")
    results = []
    for d in (clean, dirty, flagged):
        d = {n: None if y is None else (y.clone().requires_grad_() if n in NAMES else y) for n, y in d.items()}
        o, s = ours(**d, normalize=True)
        grads = torch.autograd.grad((o[:, cut:].float().square().sum(), s.square().sum()), [d[n] for n in NAMES])
        results.append([o[:, cut:], s] + [y[:, cut:] for y in grads[:5]])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.isfinite(a).all() and torch.equal(a, b)
    state = dirty["state"].clone()
    a = gated_delta_step(*(clean[n][:, cut] for n in NAMES[:5]), state, x["reset"][:, cut].cuda(), normalize=True)
    assert torch.isfinite(a).all() and torch.isfinite(state).all()
    # and no gradient flows back over it
    d = {n: (y.clone().requires_grad_() if n in NAMES else y) for n, y in clean.items()}
    o, s = ours(**d, normalize=True)
    grads = torch.autograd.grad((o[:, cut:].sum(), s.sum()), [d[n] for n in NAMES])
    assert all(not y[:, :cut].any() for y in grads[:5]) and not grads[5].any() and not grads[3][:, cut].any()


def test_every_token_resets_and_none_does():
    x = inputs(2, 40, 1, 2, 32, 32, torch.float32, seed=21)
    x["reset"][:] = True
    check_train(x, normalize=True)
    x["reset"][:] = False
    check_train(x, normalize=True)


def test_repeated_keys_full_strength():
    """An environment that stands still: one key, beta 1, no decay. Products of powers of the
    matrix inside a chunk would reach 6e3 here; the substitution keeps every digit."""
    x = inputs(1, 96, 1, 1, 64, 64, torch.float32, seed=2, resets=0.0)
    x["k"][:] = x["k"][:, :1].clone()
    x["beta"][:] = 1.0
    x["g"][:] = 0.0
    check_train(x, normalize=True)


def test_strong_decay_keeps_the_digits_of_what_follows():
    """One token of g = -100 and slow decay after it: differences of sums near 100."""
    x = inputs(1, 64, 1, 1, 32, 32, torch.float32, seed=4, resets=0.0)
    x["g"][:] = -0.01
    x["g"][:, [5, 11, 40]] = -100.0
    check_train(x, normalize=True)


def test_gradients_against_differences():
    """Central differences of the kernel's own fp32 outputs in 12 random directions. With step h
    the difference's error is h^2 of the third derivative (about 1e-4 here) plus the outputs'
    rounding over 2 h (1e-6 / 2e-2)."""
    from zeno_amd.memory import gated_delta as ours

    x = on_gpu(inputs(2, 40, 1, 2, 16, 24, torch.float32, seed=8, resets=0.05))
    r = torch.Generator(device="cuda").manual_seed(1)
    wo = torch.randn(2, 40, 2, 24, generator=r, device="cuda") / 40
    ws = torch.randn(2, 2, 16, 24, generator=r, device="cuda") / 40

    def value(d):
        o, s = ours(**d, normalize=True)
        return (o.double() * wo).sum() + (s.double() * ws).sum()

    d = {n: (y.clone().requires_grad_() if n in NAMES else y) for n, y in x.items()}
    grads = torch.autograd.grad(value(d), [d[n] for n in NAMES])
    h = 1e-2
    for n, grad in zip(NAMES, grads):
        for _ in range(2):
            way = torch.randn(grad.shape, generator=r, device="cuda")
            way /= way.norm()
            with torch.no_grad():
                slope = (value(dict(x, **{n: x[n] + h * way})) - value(dict(x, **{n: x[n] - h * way}))) / (2 * h)
            assert abs(float((grad.double() * way).sum() - slope)) < 2e-4 * max(1.0, float(grad.norm())), n


def test_results_are_reproducible_and_follow_the_stream():
    from zeno_amd.memory import gated_delta as ours

    x = on_gpu(inputs(16, 100, 2, 6, 64, 64, torch.bfloat16, seed=6))
    outs = []
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side, side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            d = {n: (y.clone().requires_grad_() if n in NAMES else y) for n, y in x.items()}
            o, s = ours(**d, normalize=True)
            outs.append([o, s, *torch.autograd.grad((o.float().square().sum(), s.sum()), [d[n] for n in NAMES])])
        stream.synchronize()
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_step_in_a_graph():
    """A captured step advances the state on every replay as the eager one does."""
    from zeno_amd.memory import gated_delta_step

    x = on_gpu(inputs(32, 1, 2, 2, 64, 64, torch.float32, seed=13))
    token = [x[n][:, 0] for n in NAMES[:5]]
    state, eager = x["state"].clone(), x["state"].clone()
    out = torch.empty_like(token[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_delta_step(*token, state.clone(), x["reset"][:, 0], normalize=True, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gated_delta_step(*token, state, x["reset"][:, 0], normalize=True, out=out)
    state.copy_(x["state"])
    for _ in range(4):
        graph.replay()
        want = gated_delta_step(*token, eager, x["reset"][:, 0], normalize=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, eager)


def test_refusals():
    from zeno_amd.memory import gated_delta as ours, gated_delta_step

    x = on_gpu(inputs(2, 4, 2, 4, 8, 8, torch.float32, seed=1))
    ok = ours(**x)
    assert ok[0].shape == (2, 4, 4, 8)
    for change, error in [({"v": x["v"][:, :, :3]}, ValueError), ({"k": x["k"].half()}, TypeError), ({"g": x["g"].double()}, TypeError),
                          ({"beta": x["beta"][:, :3]}, ValueError), ({"reset": x["reset"].int()}, TypeError),
                          ({"state": x["state"].half()}, TypeError), ({"state": x["state"][:1]}, ValueError),
                          ({"q": x["q"][:, :0], "k": x["k"][:, :0], "v": x["v"][:, :0], "g": x["g"][:, :0], "beta": x["beta"][:, :0],
                            "reset": None}, ValueError),
                          ({"g": x["g"].cpu()}, ValueError), ({"scale": float("nan")}, ValueError)]:
        with pytest.raises(error):
            ours(**dict(x, **change))
    big = on_gpu(inputs(1, 2, 1, 1, 129, 8, torch.float32, seed=1))
    with pytest.raises(ValueError, match="1 to 128"):
        ours(**big)
    token = [x[n][:, 0] for n in NAMES[:5]]
    with pytest.raises(ValueError, match="contiguous"):
        gated_delta_step(*token, x["state"].mT.contiguous().mT)
    with pytest.raises(ValueError, match="out must be"):
        gated_delta_step(*token, x["state"], out=torch.empty(1, device="cuda"))


# (batch, length, key heads, value heads, key_dim, value_dim): few heads and long axes, cut into
# segments, the last of them partial
LONG = [(1, 800, 1, 1, 64, 64), (1, 1111, 1, 2, 40, 100), (2, 770, 1, 1, 128, 128), (1, 900, 2, 2, 100, 33), (2, 800, 1, 2, 64, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_sequences(shape, dtype):
    x = inputs(*shape, dtype, seed=sum(shape), resets=0.003)
    x["g"] *= 0.05  # states that reach over several segments
    check_train(x, normalize=True)


def test_long_sequence_without_state_and_one_reset_in_a_segment():
    x = inputs(1, 1500, 1, 1, 32, 64, torch.float32, seed=31, resets=0.0)
    x["g"] *= 0.01
    x["state"] = None
    x["reset"][:, 700] = True
    check_train(x, normalize=True)


def test_nothing_passes_a_reset_between_segments():
    """NaN in one segment, cleared in a later one: the matrices over segments are cleared too."""
    from zeno_amd.memory import gated_delta as ours

    x = on_gpu(inputs(1, 2000, 1, 1, 64, 64, torch.float32, seed=12, resets=0.0))
    x["reset"][:, 1300] = True
    clean = {n: y.clone() for n, y in x.items()}
    for at, n in ((3, "v"), (260, "k"), (520, "q"), (780, "g"), (1290, "beta")):
        x[n][:, at] = float("nan")
    results = []
    for d in (clean, x):
        d = {n: (y.clone().requires_grad_() if n in NAMES else y) for n, y in d.items()}
        o, s = ours(**d, normalize=True)
        grads = torch.autograd.grad((o[:, 1300:].square().sum(), s.square().sum()), [d[n] for n in NAMES[:5]])
        results.append([o[:, 1300:], s, *(y[:, 1300:] for y in grads)])
    for a, b in zip(*results):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("advanced", ["last", "state"])
def test_a_state_advanced_before_the_backward_pass_is_noticed(advanced):
    """Steps write the state in place, outside of torch: gradients that would read it are refused."""
    from zeno_amd.memory import gated_delta as ours, gated_delta_step

    x = torch.randn(2, 9, 3, 16, device="cuda")
    g = torch.zeros(2, 9, 3, device="cuda")
    beta = torch.full_like(g, 0.5).requires_grad_()
    state = torch.randn(2, 3, 16, 16, device="cuda")
    o, last = ours(x, x, x, g, beta, state=state, normalize=True)
    token = x[:, 0], x[:, 0], x[:, 0], g[:, 0], beta[:, 0].detach()
    gated_delta_step(*token, last.detach() if advanced == "last" else state, normalize=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
