"""Results of the policy operators at places beyond 2^31 elements: wide rows of one buffer, of which every result
is a slice, written through the C entry points, against the same calls into tensors of their own."""
import ctypes as C

import pytest
import torch

from tests.policy_reference import assert_near, work_error

pytestmark = pytest.mark.gpu
S3 = C.c_int64 * 3


def far(shape, tokens, buffer, at):
    """A view of shape [B, tokens, heads, dim] (or [B, heads, dim] and others along `tokens`) whose step along
    dimension `tokens` is the buffer's row and which begins at column `at`."""
    stride, step = [0] * len(shape), 1
    for i in reversed(range(len(shape))):
        if i == tokens:
            stride[i] = buffer.stride(0)
        else:
            stride[i], step = step, step * shape[i]
    y = buffer.as_strided(shape, stride, at)
    assert at + step <= buffer.shape[1] and stride[tokens] * (shape[tokens] - 1) > 1 << 31
    return y


def rows(n, dtype):
    """So many rows in more than 2^31 elements."""
    return torch.zeros(n, (1 << 31) // (n - 2) + 8, dtype=dtype, device="cuda")


def strides(x):
    return S3(*x.stride()[:3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("b, t, hk, hv, dk, dv, along, g", [(2, 40, 2, 2, 32, 48, 1, -0.1), (2, 150, 1, 4, 40, 33, 1, -0.1), (4, 33, 2, 2, 64, 64, 0, -0.1), (2, 40, 1, 2, 24, 24, 1, 3.0),
                                                            (1030, 20, 1, 1, 64, 64, 0, -0.1)], ids=str)
def test_linear_attention(b, t, hk, hv, dk, dv, along, g, dtype):
    """In chunks and token by token (heads that grow fast), of heads that share keys, in waves of both widths, with the batch and with
    the tokens far apart."""
    from zeno_amd import _lib, memory

    lib, r = _lib.load(), torch.Generator(device="cuda").manual_seed(t)

    def normal(*s):
        return torch.randn(*s, generator=r, device="cuda").to(dtype)

    x = [normal(b, t, hk, dk), normal(b, t, hk, dk), normal(b, t, hv, dv)]
    d_o, decays = normal(b, t, hv, dv), torch.full((hv,), g, device="cuda")
    if g > 0:
        x[1] *= 2.0 ** -10
    reset = torch.zeros(b, t, dtype=torch.bool, device="cuda")
    reset[:, ::10] = True
    leaves = [y.clone().requires_grad_() for y in x]
    o, last = memory.linear_attention(*leaves, decays, reset)
    want = [o.detach(), *torch.autograd.grad(o, leaves, d_o)]
    buffer = rows((b, t)[along], dtype)
    got, at = [], 8
    for y in want:
        got.append(far(y.shape, along, buffer, at))
        at += y.numel() // y.shape[along] + 3
    a = memory._linear_inputs(*x, decays, reset, None, None, False)
    state = torch.empty_like(last)
    saved = torch.empty(max(lib.zeno_amd_linear_saved_bytes(a), 16), dtype=torch.uint8, device="cuda")
    space = torch.empty(max(lib.zeno_amd_linear_workspace_bytes(a, 0), lib.zeno_amd_linear_workspace_bytes(a, 1), 16), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.zeno_amd_linear_forward(a, got[0].data_ptr(), strides(got[0]), state.data_ptr(), saved.data_ptr(), space.data_ptr(), stream) == 0, _lib.last_error()
    grads = _lib.ZenoAmdLinearGradients(d_o=d_o.data_ptr(), d_o_stride=strides(d_o), d_q=got[1].data_ptr(), d_k=got[2].data_ptr(), d_v=got[3].data_ptr(),
                                        d_q_stride=strides(got[1]), d_k_stride=strides(got[2]), d_v_stride=strides(got[3]))
    assert lib.zeno_amd_linear_backward(a, saved.data_ptr(), grads, space.data_ptr(), stream) == 0, _lib.last_error()
    assert torch.equal(state, last)
    for n, p, w in zip(("o", "d_q", "d_k", "d_v"), got, want):
        assert torch.isfinite(w).all() and torch.equal(p, w), n
        p.zero_()
    assert not buffer.any()  # nothing beside them


def test_shared_heads_gradients_behind_2_31_parts():
    """Four value heads' parts of a long sequence's gradients of 128 keys: 2^31 floats and more, of q and of k each."""
    from zeno_amd.memory import linear_attention

    t, part = (1 << 22) + 70, 100
    r = torch.Generator(device="cuda").manual_seed(2)

    def normal(*s):
        return torch.randn(*s, generator=r, device="cuda", dtype=torch.float16)

    q, k, v, d_o = normal(1, t, 1, 128), normal(1, t, 1, 128), normal(1, t, 4, 2), normal(1, t, 4, 2)
    g = torch.tensor([-1.0, -0.7, -0.5, -2.0], device="cuda")
    reset = torch.zeros(1, t, dtype=torch.bool, device="cuda")
    reset[0, t - part] = True
    d_o[:, :t - part] = 0
    leaves = [x.requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(linear_attention(*leaves, g, reset)[0], leaves, d_o)
    tail = [x.detach()[:, t - part:].clone().requires_grad_() for x in leaves]
    want = torch.autograd.grad(linear_attention(*tail, g)[0], tail, d_o[:, t - part:].clone())
    for n, p, w in zip("qkv", got, want):
        assert_near(p[:, t - part:], w, 2 * 2.0 ** -11 + 2 * work_error(part // 32 + 32, 128, 2), "gradient of " + n)
        assert not p[:, :t - part].any(), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_linear_attention_step(dtype):
    """Outputs far apart, and a state of more than 2^31 values."""
    from zeno_amd.memory import linear_attention_step

    r = torch.Generator(device="cuda").manual_seed(3)
    b = (1 << 17) + 3
    q, k, v = (torch.randn(b, 1, 128, generator=r, device="cuda").to(dtype) for _ in range(3))
    g, state = torch.tensor([-0.1], device="cuda"), torch.zeros(b, 1, 128, 128, device="cuda")
    state[-5:] = torch.randn(5, 1, 128, 128, generator=r, device="cuda")
    few = state[-5:].clone()
    assert state.numel() > 1 << 31
    want = linear_attention_step(q[-5:], k[-5:], v[-5:], g, few)
    buffer = rows(5, dtype)
    out = far((5, 1, 128), 0, buffer, 8)
    kept = state[-5:].clone()
    assert linear_attention_step(q[-5:], k[-5:], v[-5:], g, kept, out=out) is out
    assert torch.equal(out, want) and torch.equal(kept, few)
    assert torch.equal(linear_attention_step(q, k, v, g, state)[-5:], want)
    assert torch.equal(state[-5:], few)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(40, 1, 1, 64), (3, 20, 1, 1000), (3, 2, 20, 100), (5, 1, 1, 9000)], ids=str)
def test_layer_norm(shape, dtype):
    """Rows along one dimension and along three, part of a wave, a wave and a workgroup to the row."""
    from zeno_amd import _lib, norm

    lib, r = _lib.load(), torch.Generator(device="cuda").manual_seed(4)
    x, z, d_y, d_sum = (torch.randn(shape, generator=r, device="cuda").to(dtype) for _ in range(4))
    w, b = (torch.randn(shape[-1], generator=r, device="cuda") for _ in range(2))
    leaves = [y.clone().requires_grad_() for y in (x, w, b, z)]
    y, total = norm.layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3])
    d_x, d_w, d_b, d_z = torch.autograd.grad((y, total), leaves, (d_y, d_sum))
    assert torch.equal(d_x, d_z)
    along = max(range(3), key=lambda i: shape[i])
    buffer = rows(shape[along], dtype)
    got, at = [], 8
    for i in range(3):
        got.append(far(shape, along, buffer, at))
        at += x.numel() // shape[along] + 3
    stream = torch.cuda.current_stream().cuda_stream
    a = norm._inputs(x, z, w, b, 1e-5)
    assert lib.zeno_amd_norm_forward(a, got[0].data_ptr(), strides(got[0]), got[1].data_ptr(), strides(got[1]), stream) == 0, _lib.last_error()
    a = norm._inputs(got[1], None, w, b, 1e-5)  # the sum, read where it was written
    weights = [torch.empty_like(w), torch.empty_like(b)]
    space = torch.empty(lib.zeno_amd_norm_workspace_bytes(a), dtype=torch.uint8, device="cuda")
    grads = _lib.ZenoAmdNormGradients(d_y.data_ptr(), d_sum.data_ptr(), got[2].data_ptr(), weights[0].data_ptr(), weights[1].data_ptr(), strides(d_y), strides(d_sum), strides(got[2]))
    assert lib.zeno_amd_norm_backward(a, grads, space.data_ptr(), stream) == 0, _lib.last_error()
    for n, p, want in zip(("y", "sum", "d_x", "d_weight", "d_bias"), got + weights, (y, total, d_x, d_w, d_b)):
        assert torch.equal(p, want), n
    for p in got:
        p.zero_()
    assert not buffer.any()
