"""The orthogonalisation's argument checks, which come before any GPU work."""
import pytest
import torch

from zeno_amd import _lib, optim


def args(**change):
    a = dict(dtype=0, count=1, rows=8, cols=8, steps=5, a=3.4445, b=-4.7750, c=2.0315, eps=1e-7, x=256, out=256)
    return _lib.ZenoAmdOrthogonalize(**{**a, **change})


@pytest.mark.parametrize("change, words", [
    ({"dtype": 3}, "dtype"), ({"count": 0}, "positive"), ({"rows": 0}, "positive"), ({"cols": 1 << 17}, "65536"), ({"count": 1 << 16}, "65535"),
    ({"steps": 0}, "steps"), ({"steps": 101}, "steps"), ({"eps": 0.0}, "eps"), ({"a": float("inf")}, "finite"), ({"x": None}, "null"),
    ({"a": 3.0, "b": 1.0, "c": 1.0}, "grow")])
def test_refused(change, words):
    lib = _lib.load()
    assert lib.zeno_amd_orthogonalize(args(**change), 256, None) == -6
    assert words in _lib.last_error()
    assert lib.zeno_amd_orthogonalize_workspace_bytes(args(**change)) == 0


def test_workspace():
    lib = _lib.load()
    assert lib.zeno_amd_orthogonalize_workspace_bytes(args()) > 0
    assert lib.zeno_amd_orthogonalize(args(), None, None) == -6
    assert lib.zeno_amd_orthogonalize(args(), 8, None) == -6
    assert lib.zeno_amd_orthogonalize(None, 256, None) == -6


def test_python_refuses():
    with pytest.raises(ValueError, match="GPU"):
        optim.orthogonalize(torch.zeros(2, 3))
    with pytest.raises(TypeError):
        optim.orthogonalize(torch.zeros(2, 3, dtype=torch.float64))
