"""What torch's tracers record of the operators on torch tensors. The library's calls are no torch operations: a
recording of those alone has the memory that a call allocates, and nothing that writes it. (No GPU: the library's
calls do nothing here.)"""
import contextlib

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from zeno_amd import _torch, memory, norm, optim

Q, G, STATE = torch.randn(2, 4, 1, 8), torch.zeros(1), torch.zeros(2, 1, 8, 8)
WHOLE = {"linear_attention": lambda q: memory.linear_attention(q, q, q, G)[0], "gated_delta": lambda q: memory.gated_delta(q, q, q, q[..., 0], q[..., 0])[0],
         "layer_norm": lambda q: norm.layer_norm(q), "layer_norm with a stream": lambda q: norm.layer_norm(q, residual=q)[1], "rows along five dimensions": lambda q: norm.layer_norm(q[None])}
IN_PLACE = {"linear_attention_step": lambda q: memory.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], G, STATE),
            "gated_delta_step": lambda q: memory.gated_delta_step(q[:, 0], q[:, 0], q[:, 0], q[:, 0, :, 0], q[:, 0, :, 0], STATE),
            "orthogonalize": lambda q: optim.orthogonalize(q[:, :, 0])}


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """The names of the library's calls; the checks of operands take what is not on the GPU."""
    made = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: made.append(name) or 0

    real_on = _torch.on
    for m in (memory, norm, optim):
        monkeypatch.setattr(m.L, "load", Library)
        if hasattr(m, "_check"):
            monkeypatch.setattr(m, "_check", lambda *a: None)
        if hasattr(m, "stream"):
            monkeypatch.setattr(m, "stream", lambda x: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)  # the device of tensors here has no number
    assert isinstance(real_on(Q), contextlib.nullcontext)
    return made


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", WHOLE)
def test_traced_as_calls(name, calls):
    """With gradients wanted and without: the trace holds the call, and running it makes the library's."""
    for wanted in (False, True):
        for grad in (torch.enable_grad, torch.no_grad):
            with grad():
                traced = torch.jit.trace(WHOLE[name], Q.clone().requires_grad_(wanted), check_trace=False)
            assert "prim::PythonOp" in [n.kind() for n in traced.graph.nodes()], (wanted, grad)
            calls.clear()
            traced(Q)
            assert any("forward" in c for c in calls), (wanted, grad)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", IN_PLACE)
def test_what_a_trace_would_lose_is_refused(name, calls):
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(IN_PLACE[name], Q, check_trace=False)
    assert not calls


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("options", [{}, {"pre_dispatch": True}], ids=str)
@pytest.mark.parametrize("name", [*WHOLE, *IN_PLACE])
def test_graphs_of_torch_operations_are_refused(name, options, calls):
    for grad in (torch.enable_grad, torch.no_grad):
        with grad(), pytest.raises(RuntimeError, match="graph of those"):
            make_fx({**WHOLE, **IN_PLACE}[name], **options)(Q)
    assert not any("forward" in c or "step" in c or c.endswith("orthogonalize") for c in calls)


def test_other_modes_are_none_of_that(calls):
    """Modes that look at operations and do not record them change nothing."""
    from torch.utils.flop_counter import FlopCounterMode

    with torch.device("cpu"), FlopCounterMode(display=False):
        for f in WHOLE.values():
            f(Q)
    assert sum("forward" in c for c in calls) == len(WHOLE)
