"""The gated delta rule refuses sizes that a launch cannot take (2^32 threads) before anything is
enqueued."""
import ctypes as C

import pytest

from zeno_amd import _lib


def args(**change):
    a = dict(dtype=2, batch=1, length=1, key_heads=1, value_heads=1, key_dim=128, value_dim=128, normalize=1, scale=1.0, q=16, k=16, v=16, g=16, beta=16)
    return _lib.ZenoAmdDeltaInputs(**{**a, **change})


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("sizes, threads", [(dict(key_dim=128, value_dim=128), 512), (dict(key_dim=8, value_dim=65), 512), (dict(key_dim=64, value_dim=64), 256)])
def test_sequences(lib, sizes, threads):
    most = (1 << 32) // threads - 1
    strides = (C.c_int64 * 3)()
    assert lib.zeno_amd_delta_saved_bytes(args(batch=most, length=33, **sizes)) > 0
    assert lib.zeno_amd_delta_saved_bytes(args(batch=most + 1, length=33, **sizes)) == 0
    for change in (dict(batch=most + 1, length=33), dict(batch=(most + 1) // 8, value_heads=8, length=2)):
        assert lib.zeno_amd_delta_forward(args(**change, **sizes), 16, strides, 16, None, None, None) == -6
        assert "too many sequences" in _lib.last_error()
        grad = _lib.ZenoAmdDeltaGradients(d_o=16, d_q=16, d_k=16, d_v=16, d_g=16, d_beta=16)
        assert lib.zeno_amd_delta_backward(args(**change, **sizes), 16, 16, grad, 16, None) == -6
        assert "too many sequences" in _lib.last_error()


@pytest.mark.parametrize("sizes, waves", [(dict(key_dim=128, value_dim=128), 4), (dict(key_dim=32, value_dim=128), 4), (dict(key_dim=64, value_dim=128), 2)])
def test_steps(lib, sizes, waves):
    heads = (1 << 26) // waves
    for change in (dict(batch=heads), dict(batch=heads // 4, value_heads=4)):
        assert lib.zeno_amd_delta_step(args(**change, **sizes), 16, (C.c_int64 * 3)(), 16, None) == -6
        assert "too many sequences" in _lib.last_error()


@pytest.mark.gpu
def test_the_sum_over_shared_heads_of_more_than_2_to_28_values():
    """The last sequences of a large batch have the gradients that they have alone."""
    import torch

    from zeno_amd.memory import gated_delta

    r = torch.Generator(device="cuda").manual_seed(1)
    batch, length, few = 137500, 16, 64
    q, k = (torch.randn(batch, length, 1, 128, generator=r, device="cuda", dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    assert q.numel() > 1 << 28
    v = torch.randn(batch, length, 2, 8, generator=r, device="cuda", dtype=torch.bfloat16)
    g, beta = -torch.rand(batch, length, 2, generator=r, device="cuda"), torch.rand(batch, length, 2, generator=r, device="cuda")
    grads = torch.autograd.grad(gated_delta(q, k, v, g, beta, normalize=True)[0], (q, k), v)
    q2, k2 = (x[-few:].detach().requires_grad_() for x in (q, k))
    alone = torch.autograd.grad(gated_delta(q2, k2, v[-few:], g[-few:], beta[-few:], normalize=True)[0], (q2, k2), v[-few:])
    for a, b in zip(grads, alone):
        assert torch.equal(a[-few:], b) and b.any()
