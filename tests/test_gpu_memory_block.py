"""A policy's block of linear attention and norms, as they are used together: the features and their
stream normalised, projected, remembered, each head's output normalised, projected and added to the
stream, which is normalised again; whole sequences with gradients, token by token, and in a graph.

Tolerances: each of the block's stages adds errors as its own tests have them (`tolerance`, the longest chain
being the features' or the attention's). The norm of the heads' outputs divides a row by its spread, and so
makes the errors of what came before larger by the size of the row's terms against that spread (`gain`, from
the definition), once in the outputs and once more in their gradients, in which the row's spread stands again.
"""
import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.linear_reference import linear_attention as exact_attention
from tests.norm_reference import layer_norm as exact_norm
from tests.policy_reference import assert_near, work_error

pytestmark = pytest.mark.gpu
WIDE, HEADS, KEY, VALUE = 96, 2, 16, 24
STAGES = 7  # two sums and norms, two projections, the attention, its features and the heads' norm


def operands(b, t, seed):
    r = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=r)

    return {"x": normal(b, t, WIDE), "stream": normal(b, t, WIDE), "w1": 1 + 0.2 * normal(WIDE), "b1": 0.1 * normal(WIDE), "in": normal(WIDE, HEADS * (2 * KEY + VALUE)) / WIDE ** 0.5,
            "g": -torch.exp(torch.linspace(-3.0, 0.0, HEADS)), "state": torch.rand(b, HEADS, KEY, VALUE, generator=r), "wh": 1 + 0.2 * normal(VALUE), "bh": 0.1 * normal(VALUE),
            "out": normal(HEADS * VALUE, WIDE) / (HEADS * VALUE) ** 0.5, "w2": 1 + 0.2 * normal(WIDE), "b2": 0.1 * normal(WIDE), "reset": torch.rand(b, t, generator=r) < 0.1}


LEAVES = [n for n in operands(1, 1, 0) if n != "reset"]


def heads_of(y, project):
    """Positive features, as linear attention is used: no product of two of them cancels."""
    q, k, v = (y @ project).split([HEADS * KEY, HEADS * KEY, HEADS * VALUE], -1)
    q, k = torch.nn.functional.softplus(q), torch.nn.functional.softplus(k)
    return q.unflatten(-1, (HEADS, KEY)), k.unflatten(-1, (HEADS, KEY)), v.unflatten(-1, (HEADS, VALUE))


def block(p, norm, attend):
    y, stream = norm(p["x"], p["w1"], p["b1"], residual=p["stream"])
    tokens = heads_of(y, p["in"])
    o, last = attend(*tokens, p["g"], p["reset"], p["state"])
    y, stream = norm(norm(o, p["wh"], p["bh"]).flatten(-2) @ p["out"], p["w2"], p["b2"], residual=stream)
    return (y, stream, last), tokens, o


def gain(p, tokens, o):
    """The terms of a head's output by their size, against the spread of its row."""
    sizes, _ = exact_attention(*(z.detach().abs() for z in tokens), p["g"].detach(), p["reset"], p["state"].detach().abs())
    spread = o.detach().std(-1, correction=0)
    return float((sizes.norm(dim=-1) / VALUE ** 0.5 / spread).max())


@pytest.mark.parametrize("b, t", [(3, 1), (5, 40), (1, 400)])
def test_sequences_and_gradients(b, t):
    from zeno_amd.memory import linear_attention
    from zeno_amd.norm import layer_norm

    x = operands(b, t, seed=b + t)
    ref = {n: y.double().requires_grad_() if n in LEAVES else y for n, y in x.items()}
    dev = {n: y.cuda().requires_grad_(n in LEAVES) for n, y in x.items()}
    want, tokens, o = block(ref, lambda s, w, c, residual=None: exact_norm(s, w, c, residual), exact_attention)
    got, _, _ = block(dev, layer_norm, linear_attention)
    grown = max(gain(ref, tokens, o), 1.0)
    assert grown < 10
    each = work_error(max(t // 32 + 32 + KEY + VALUE, WIDE))
    r = torch.Generator().manual_seed(1)
    down = [torch.randn(y.shape, generator=r) for y in want]
    grads = torch.autograd.grad(want, [ref[n] for n in LEAVES], [d.double() for d in down])
    ours = torch.autograd.grad(got, [dev[n] for n in LEAVES], [d.cuda() for d in down])
    for n, p, q in zip(("y", "stream", "last"), got, want):
        assert_near(p, q, STAGES * grown * each, n)
    for n, p, q in zip(LEAVES, ours, grads):
        assert_near(p, q, 2 * STAGES * grown ** 2 * each, "gradient of " + n)


def test_token_by_token():
    """A block stepped along with the environments: the sequence's results."""
    from zeno_amd.memory import linear_attention, linear_attention_step
    from zeno_amd.norm import layer_norm

    x = operands(64, 20, seed=2)
    ref = {n: y.double() if n in LEAVES else y for n, y in x.items()}
    _, tokens, o = block(ref, lambda s, w, c, residual=None: exact_norm(s, w, c, residual), exact_attention)
    grown, dev = max(gain(ref, tokens, o), 1.0), {n: y.cuda() for n, y in x.items()}
    (y, stream, last), _, _ = block(dev, layer_norm, linear_attention)
    state, ys, streams = dev["state"].clone(), [], []
    for t in range(20):
        def step(q, k, v, g, reset, s):
            return linear_attention_step(q, k, v, g, s, reset), s

        (a, b, _), _, _ = block({**dev, "x": dev["x"][:, t], "stream": dev["stream"][:, t], "reset": dev["reset"][:, t], "state": state}, layer_norm, step)
        ys.append(a), streams.append(b)
    tol = 2 * STAGES * grown * work_error(WIDE)
    assert_near(torch.stack(ys, 1), y, tol, "y")
    assert_near(torch.stack(streams, 1), stream, tol, "stream")
    assert_near(state, last, tol, "state")


@pytest.mark.parametrize("t", [24, 200])
def test_captured_and_replayed(t):
    """The block with its gradients in a graph, replayed with other inputs and eager work between: the eager results."""
    from zeno_amd.memory import linear_attention
    from zeno_amd.norm import layer_norm

    x = {n: y.cuda() for n, y in operands(2, t, seed=6).items()}
    down = None

    def run(z):
        nonlocal down
        leaves = {n: y.detach().requires_grad_(n in LEAVES) for n, y in z.items()}
        out, _, _ = block(leaves, layer_norm, linear_attention)
        if down is None:
            down = [torch.randn_like(y) for y in out]
        grads = torch.autograd.grad(out, [leaves[n] for n in LEAVES], down)
        return [y.detach() for y in out] + list(grads)

    held, side = {n: y.clone() for n, y in x.items()}, torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(held)
    for i in range(4):
        for n in LEAVES:
            if n != "g":
                held[n].copy_(x[n] * (1 + i / 8))
        eager = run(held)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), i


def test_tangents_are_refused():
    """Forward-mode differentiation, which the operators do not have, is an error and no result without a tangent."""
    import torch.autograd.forward_ad as forward

    from zeno_amd.memory import linear_attention
    from zeno_amd.norm import layer_norm

    q = torch.randn(1, 4, 1, 8, device="cuda")
    with forward.dual_level():
        dual = forward.make_dual(q, torch.ones_like(q))
        with pytest.raises(RuntimeError):
            linear_attention(dual, q, q, torch.zeros(1, device="cuda"))
        with pytest.raises(RuntimeError):
            layer_norm(dual)
    assert torch.isfinite(layer_norm(q)).all()


def test_the_example_with_linear_attention():
    spec = importlib.util.spec_from_file_location("memory_policy", Path(__file__).resolve().parents[1] / "examples" / "memory_policy.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    history, apart = example.train(envs=200, updates=4, length=40, log=lambda line: None, memory="linear")
    assert len(history) == 4 and np.isfinite(history).all()
    # What was acted token by token is what the training pass differentiates: chains of 40 tokens, 32 dimensions and a projection's
    # 64, whose terms are at most a dozen times the largest output.
    assert apart < 12 * (40 + 32 + 64) * 2.0 ** -24
