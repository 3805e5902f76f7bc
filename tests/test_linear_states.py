"""``linear`` under torch's tracer: recorded as a call that computes, with the sizes of the tensors it is given."""
from __future__ import annotations

import contextlib

import pytest
import torch

from mintext_amd import _lib as L
from mintext_amd.kernels import linear


@pytest.fixture
def launches(monkeypatch):
    """The calls of entry points, with their arguments, that would be made on a device."""
    made = []
    monkeypatch.setattr(L, "require_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(L, "on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(L, "stream", lambda d: 0)
    monkeypatch.setattr(L, "call", lambda *a: made.append(a))
    return made


FORMS = {
    "plain": lambda t, w, b: linear(t, w),
    "bias": lambda t, w, b: linear(t, w, b, activation="silu"),
    "residual": lambda t, w, b: linear(t, w, b, activation="gelu", residual=t[..., :5].contiguous()),
}


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_a_trace_records_the_call(launches, form, grad):
    w, b = torch.randn(8, 5).requires_grad_(grad), torch.randn(5)
    traced = torch.jit.trace(FORMS[form], (torch.randn(4, 8), w, b), check_trace=False)
    launches.clear()
    out = traced(torch.randn(7, 8), w, b)
    assert out.shape == (7, 5) and out.requires_grad == grad
    (call,) = launches
    assert call[0] == "mtx_linear" and call[6:9] == (7, 8, 5)  # the sizes of this call, not of the traced one


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("form", FORMS)
def test_a_trace_computes(dev, form):
    w, b = torch.randn(8, 5, device=dev), torch.randn(5, device=dev)
    x, y = torch.randn(4, 8, device=dev), torch.randn(7, 8, device=dev)
    traced = torch.jit.trace(FORMS[form], (x, w, b), check_trace=False)
    assert torch.equal(traced(y, w, b), FORMS[form](y, w, b))
