"""Outputs of the policy operators that overlap themselves or what a call reads are refused before
anything is enqueued; views of one buffer are not taken for that."""
import ctypes as C

import pytest
import torch

from zeno_amd import _lib

MIB = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def token(**change):
    """One token of 4 sequences, two heads of 32 x 64, every array in a MiB of its own."""
    a = dict(dtype=0, batch=4, length=1, key_heads=2, value_heads=2, key_dim=32, value_dim=64, normalize=1, scale=1.0, q=MIB, k=2 * MIB, v=3 * MIB,
             g=4 * MIB, beta=5 * MIB, q_stride=(64, 0, 32), k_stride=(64, 0, 32), v_stride=(128, 0, 64), g_stride=(2, 0, 1), beta_stride=(2, 0, 1))
    return _lib.ZenoAmdDeltaInputs(**{**a, **change})


@pytest.mark.parametrize("o, stride, change, words", [
    (MIB, (128, 0, 64), {}, "overlaps an input"),                               # q
    (2 * MIB + 1023, (128, 0, 64), {}, "overlaps an input"),                    # k's last byte
    (3 * MIB + 256, (128, 0, 64), {}, "overlaps v"),                            # v, but not in its place
    (3 * MIB, (64, 0, 256), {}, "overlaps v"),                                  # v in another order
    (5 * MIB - 128, (128, 0, 64), {}, "overlaps an input"),                     # beta
    (7 * MIB, (0, 0, 64), {}, "overlaps itself"), (7 * MIB, (128, 0, 0), {}, "overlaps itself"), (7 * MIB, (96, 0, 64), {}, "overlaps itself"),
    (7 * MIB, (128, 0, 64), {"reset": 7 * MIB + 4, "reset_stride": (1, 0)}, "overlaps an input"),
    (6 * MIB + 1024, (128, 0, 64), {}, "overlaps the state"),
    (8 * MIB, (128, 0, 64), {"v": 6 * MIB}, "the state overlaps an input"), (8 * MIB, (128, 0, 64), {"g": 6 * MIB + 60}, "the state overlaps an input"),
    (MIB + 128, (512, 0, 128), {"q_stride": (512, 0, 64)}, "overlaps an input")])  # beside q in one buffer, but heads meet
def test_a_step_refuses_outputs_that_overlap(lib, o, stride, change, words):
    assert lib.zeno_amd_delta_step(token(**change), o, (C.c_int64 * 3)(*stride), 6 * MIB, None) == -6
    assert words in _lib.last_error()


def test_a_sequence_refuses_outputs_that_overlap(lib):
    a = token(length=5, q_stride=(320, 64, 32), k_stride=(320, 64, 32), v_stride=(640, 128, 64), g_stride=(10, 2, 1), beta_stride=(10, 2, 1), state=9 * MIB)
    for o, last, words in ((MIB, 6 * MIB, "overlaps an input"), (9 * MIB, 6 * MIB, "overlaps an input"), (7 * MIB, 7 * MIB, "overlaps the state"),
                           (7 * MIB, 9 * MIB + 16, "the state overlaps an input"), (7 * MIB, 2 * MIB, "the state overlaps an input")):
        assert lib.zeno_amd_delta_forward(a, o, (C.c_int64 * 3)(640, 128, 64), last, None, None, None) == -6
        assert words in _lib.last_error()


@pytest.mark.parametrize("stride", [(0, 8, 1), (64, 0, 1), (64, 8, 0), (64, 4, 1), (32, 8, 1)], ids=str)
def test_an_update_refuses_an_output_that_overlaps_itself(lib, stride):
    a = _lib.ZenoAmdOrthogonalize(dtype=0, count=2, rows=8, cols=8, steps=5, a=3.4445, b=-4.7750, c=2.0315, eps=1e-7, x=MIB, x_stride=(64, 8, 1),
                                  out=2 * MIB, out_stride=stride)
    assert lib.zeno_amd_orthogonalize(a, 4 * MIB, None) == -6
    assert "overlaps itself" in _lib.last_error()


@pytest.mark.gpu
def test_on_tensors():
    from zeno_amd.memory import gated_delta_step
    from zeno_amd.optim import orthogonalize

    r = torch.Generator(device="cuda").manual_seed(1)

    def normal(*s):
        return torch.randn(*s, generator=r, device="cuda")

    x = normal(6, 4, 2, 128)  # q, k, v and a place for o in one buffer, beside each other
    q, k, v, place = x.unbind(1)
    g, beta, state = -torch.rand(6, 2, device="cuda"), torch.rand(6, 2, device="cuda"), normal(6, 2, 128, 128)
    want_state = state.clone()
    want = gated_delta_step(q.clone(), k.clone(), v.clone(), g, beta, want_state, normalize=True)
    for out in (q, k, state[:, :, 0], want[:1].expand(6, 2, 128)):
        with pytest.raises(ValueError, match="overlaps"):
            gated_delta_step(q, k, v, g, beta, state, normalize=True, out=out)
    y = x.transpose(1, 2).contiguous()  # head by head instead
    for buffer in (x.unbind(1), y.unbind(2)):
        q, k, v, place = buffer
        for out in (place, v):
            s = state.clone()
            assert torch.equal(gated_delta_step(q, k, v, g, beta, s, normalize=True, out=out), want) and torch.equal(s, want_state)
    m = normal(40, 60)
    want = orthogonalize(m)
    with pytest.raises(ValueError, match="overlaps itself"):
        orthogonalize(m, out=m[:1].expand(40, 60))
    wide = torch.zeros(41, 60, device="cuda")
    wide[:40] = m
    assert torch.equal(orthogonalize(wide[:40], out=wide[1:]), want)  # read before it is written
