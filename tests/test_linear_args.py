"""Linear attention's C entry points refuse what they cannot take before anything is enqueued (no GPU)."""
import ctypes as C

import pytest

from zeno_amd import _lib

MIB = 1 << 20
S3 = C.c_int64 * 3
S2 = C.c_int64 * 2
KEY, VALUE = (280, 40, 20), (672, 96, 24)  # 2 sequences of 7 tokens, two key heads of 20 and four value heads of 24


def operands(**change):
    """Every array in a MiB of its own."""
    a = dict(dtype=0, batch=2, length=7, key_heads=2, value_heads=4, key_dim=20, value_dim=24, decay_gradient=1, scale=1.0, q=MIB, k=2 * MIB, v=3 * MIB, g=4 * MIB,
             reset=5 * MIB, state=6 * MIB, q_stride=KEY, k_stride=KEY, v_stride=VALUE, reset_stride=(7, 1))
    a = {**a, **change}
    for n in ("q_stride", "k_stride", "v_stride"):
        a[n] = S3(*a[n])
    a["reset_stride"] = S2(*a["reset_stride"])
    return _lib.ZenoAmdLinearInputs(**a)


def gradients(**change):
    g = dict(d_o=7 * MIB, d_o_stride=S3(*VALUE), d_last=8 * MIB, d_q=9 * MIB, d_k=10 * MIB, d_v=11 * MIB, d_g=12 * MIB, d_state=13 * MIB, d_q_stride=S3(*KEY),
             d_k_stride=S3(*KEY), d_v_stride=S3(*VALUE))
    return _lib.ZenoAmdLinearGradients(**{**g, **change})


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(rc, words):
    assert rc == -6 and words in _lib.last_error(), (rc, _lib.last_error())


def forward(lib, a, o=14 * MIB, stride=VALUE, last=15 * MIB, saved=None, workspace=16 * MIB):
    return lib.zeno_amd_linear_forward(a, o, None if stride is None else S3(*stride), last, saved, workspace, None)


def step(lib, a, o=14 * MIB, stride=VALUE, state=15 * MIB):
    return lib.zeno_amd_linear_step(a, o, None if stride is None else S3(*stride), state, None)


@pytest.mark.parametrize("change, words", [
    ({"dtype": 3}, "dtype"), ({"batch": 0}, "positive"), ({"length": 0}, "positive"), ({"key_heads": 0}, "positive"), ({"value_heads": 0}, "positive"),
    ({"value_heads": 5}, "multiple"), ({"value_heads": 1}, "multiple"), ({"key_dim": 0}, "1 to 128"), ({"key_dim": 129}, "1 to 128"), ({"value_dim": 129}, "1 to 128"),
    ({"batch": 1 << 31}, "too many"), ({"length": 1 << 31}, "too many"), ({"q": None}, "null input"), ({"k": None}, "null input"), ({"v": None}, "null input"),
    ({"g": None}, "null input"), ({"scale": float("nan")}, "scale"), ({"scale": float("-inf")}, "scale")])
def test_sizes_types_and_nulls(lib, change, words):
    a = operands(**change)
    refused(forward(lib, a), words)
    refused(lib.zeno_amd_linear_backward(a, None, gradients(), 16 * MIB, None), words)
    refused(step(lib, operands(**{"length": 1, **change})), words)


def test_null_results(lib):
    refused(forward(lib, None), "null")
    refused(forward(lib, operands(), o=None), "null")
    refused(forward(lib, operands(), stride=None), "null")
    refused(forward(lib, operands(), last=None), "null")
    refused(lib.zeno_amd_linear_backward(operands(), None, None, 16 * MIB, None), "null")
    for n in ("d_o", "d_q", "d_k", "d_v"):
        refused(lib.zeno_amd_linear_backward(operands(), None, gradients(**{n: None}), 16 * MIB, None), "null")
    refused(lib.zeno_amd_linear_backward(operands(), None, gradients(d_g=None), 16 * MIB, None), "decay_gradient")
    refused(lib.zeno_amd_linear_backward(operands(decay_gradient=0), None, gradients(), 16 * MIB, None), "decay_gradient")
    refused(step(lib, operands()), "one token")
    refused(step(lib, operands(length=1), state=None), "null")
    refused(step(lib, operands(length=1), o=None), "null")
    assert lib.zeno_amd_linear_saved_bytes(None) == lib.zeno_amd_linear_workspace_bytes(None, 1) == 0


def test_buffers(lib):
    long = operands(length=7000, q_stride=(280000, 40, 20), k_stride=(280000, 40, 20), v_stride=(672000, 96, 24), reset_stride=(7000, 1))
    refused(forward(lib, long, workspace=None), "workspace")
    refused(forward(lib, operands(), saved=17 * MIB + 8), "aligned")
    refused(forward(lib, operands(), workspace=16 * MIB + 4), "aligned")
    refused(lib.zeno_amd_linear_backward(long, None, gradients(), 16 * MIB, None), "saved")
    refused(lib.zeno_amd_linear_backward(long, 17 * MIB, gradients(), None, None), "workspace")
    refused(lib.zeno_amd_linear_backward(operands(), 17 * MIB + 4, gradients(), 16 * MIB, None), "aligned")


@pytest.mark.parametrize("change, words", [
    (dict(o=MIB), "an input"), (dict(o=2 * MIB + 100), "an input"), (dict(o=3 * MIB), "overlaps v"), (dict(o=3 * MIB - 4), "overlaps v"), (dict(o=4 * MIB), "an input"),
    (dict(o=5 * MIB + 8), "an input"), (dict(o=6 * MIB), "an input"), (dict(last=6 * MIB), "an input"), (dict(last=3 * MIB), "an input"), (dict(last=14 * MIB + 64), "the state"),
    (dict(stride=(672, 96, 23)), "itself"), (dict(stride=(0, 96, 24)), "itself"), (dict(stride=(672, 0, 24)), "itself")])
def test_results_that_overlap(lib, change, words):
    refused(forward(lib, operands(), **change), words)


@pytest.mark.parametrize("change, words", [
    (dict(o=MIB), "an input"), (dict(o=3 * MIB + 4), "overlaps v"), (dict(o=3 * MIB, stride=(700, 96, 24)), "overlaps v"), (dict(state=3 * MIB), "an input"),
    (dict(state=2 * MIB), "an input"), (dict(state=14 * MIB), "the state"), (dict(stride=(96, 96, 0)), "itself")])
def test_steps_that_overlap(lib, change, words):
    refused(step(lib, operands(length=1), **change), words)


@pytest.mark.parametrize("change, words", [
    (dict(d_q=MIB), "an input"), (dict(d_k=7 * MIB), "an input"), (dict(d_v=8 * MIB), "an input"), (dict(d_g=6 * MIB), "an input"), (dict(d_state=3 * MIB), "an input"),
    (dict(d_k=9 * MIB + 100), "gradients overlap"), (dict(d_g=11 * MIB), "gradients overlap"), (dict(d_state=12 * MIB + 8), "gradients overlap"),
    (dict(d_q_stride=S3(280, 40, 0)), "itself"), (dict(d_v_stride=S3(672, 90, 24)), "itself")])
def test_gradients_that_overlap(lib, change, words):
    refused(lib.zeno_amd_linear_backward(operands(), None, gradients(**change), 16 * MIB, None), words)


@pytest.mark.parametrize("dims, waves", [((64, 64), 9), ((64, 32), 9), ((8, 65), 20), ((128, 128), 20), ((65, 1), 20)])
def test_launches(lib, dims, waves):
    """Less than 2^32 threads, 64 to a wave, also of the gradients of one token."""
    most = ((1 << 26) - 32) // waves
    sizes = dict(length=1, key_heads=1, value_heads=1, key_dim=dims[0], value_dim=dims[1])
    for batch, heads in ((most + 1, 1), (most // 2 + 1, 2)):
        a = operands(**{**sizes, "batch": batch, "value_heads": heads})
        for rc in (forward(lib, a), step(lib, a), lib.zeno_amd_linear_backward(a, None, gradients(), 16 * MIB, None)):
            refused(rc, "too many sequences")


def test_what_is_kept(lib):
    """Between segments a state each, and with a decay that is learned its slope; nothing where one segment does."""
    kept, space = lib.zeno_amd_linear_saved_bytes, lib.zeno_amd_linear_workspace_bytes
    assert kept(operands()) == 0 and space(operands(), 0) == 0
    assert kept(operands(length=32)) == kept(operands(length=64)) == 0
    state = 4 * 20 * 24
    assert kept(operands(length=128, decay_gradient=0)) == 8 * state  # two segments of two chunks
    assert kept(operands(length=128)) == 2 * 8 * state
    assert kept(operands(batch=2000, length=128)) == 0  # enough waves without
    assert kept(operands(length=1 << 20, decay_gradient=0)) == 8 * 255 * state
    assert space(operands(key_heads=4, decay_gradient=0), 1) == 0
    assert space(operands(decay_gradient=0), 1) == 2 * 4 * 2 * 7 * 4 * 20  # q's and k's gradients by value head
