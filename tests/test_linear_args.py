"""Calls of the dense product that are refused, before anything is launched (host only)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mintext_amd import _lib as L
from mintext_amd.kernels import linear


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args, kwargs, error", [
    ((z(4, 8), z(9, 8)), {}, ValueError),                                    # K differs
    ((z(4, 8), z(2, 8, 8)), {}, ValueError),                                 # a stack of weights
    ((z(4, 8), z(8, 16), z(8)), {}, ValueError),                             # bias of another length
    ((z(4, 8), z(8, 16), z(1, 16)), {}, ValueError),
    ((z(4, 8), z(8, 16)), dict(residual=z(16)), ValueError),                 # broadcast by the caller, not here
    ((z(4, 8), z(8, 16)), dict(activation="tanh"), ValueError),
    ((z(4, 8), z(8, 16, dtype=torch.float32)), {}, TypeError),               # mixed types
    ((z(4, 8), z(8, 16), z(16, dtype=torch.float32)), {}, TypeError),
    ((z(4, 8, dtype=torch.float16), z(8, 16, dtype=torch.float16)), {}, TypeError),
    ((z(4, 8), z(8, 16)), {}, RuntimeError),                                 # no device
])
def test_refusals(args, kwargs, error):
    with pytest.raises(error):
        linear(*args, **kwargs)


def test_entry_points_refuse():
    lib = L.lib()
    buf = ctypes.create_string_buffer(1 << 20)
    d, P, n = ctypes.addressof(buf), None, 1 << 20
    ok = lambda M, K, N: lib.mtx_linear_workspace_size(M, K, N)
    assert ok(16, 8, 8) >= 0 and ok(-1, 8, 8) < 0
    call = lambda *a: lib.mtx_linear(*a)
    assert call(d, d, P, P, 2, 4, 8, 8, 0, d, P, d, n, P) == L.MTX_ERR_ARG       # dtype
    assert call(d, d, P, P, 1, 4, 8, 8, 5, d, P, d, n, P) == L.MTX_ERR_ARG       # activation
    assert call(d, d, P, P, 1, -4, 8, 8, 0, d, P, d, n, P) == L.MTX_ERR_ARG
    assert call(P, d, P, P, 1, 4, 8, 8, 0, d, P, d, n, P) == L.MTX_ERR_ARG       # no x
    assert call(d, d, P, P, 1, 4, 8, 8, 0, P, P, d, n, P) == L.MTX_ERR_ARG       # no out
    assert call(d, d, P, P, 1, 1 << 23, 8, 8, 0, d, P, d, 1 << 40, P) == L.MTX_ERR_UNSUPPORTED
    assert call(d, d, P, P, 1, 4096, 8, 8, 0, d, P, P, 0, P) == L.MTX_ERR_WORKSPACE
    back = lambda dy, x, w, pre, act, dz, dx, dw, db, ws=d, size=n, M=4: lib.mtx_linear_bwd(
        dy, x, w, pre, 1, M, 8, 8, act, dz, dx, dw, db, ws, size, P)
    assert back(d, d, d, P, 0, P, d, P, P, ws=P, size=0, M=4096) == L.MTX_ERR_WORKSPACE
    assert back(d, d, d, P, 2, d, d, d, d) == L.MTX_ERR_ARG      # an activation without z
    assert back(d, d, d, d, 2, P, d, d, d) == L.MTX_ERR_ARG      # nowhere to write dz
    assert back(d, d, d, d, 9, d, d, d, d) == L.MTX_ERR_ARG
    assert back(P, d, d, P, 0, P, d, P, P) == L.MTX_ERR_ARG      # no gradient
    assert back(d, P, d, P, 0, P, P, d, P) == L.MTX_ERR_ARG      # dw without x
    assert back(d, d, P, P, 0, P, d, P, P) == L.MTX_ERR_ARG      # dx without w
    assert back(d, d, d, P, 0, P, P, P, P) == L.MTX_OK           # nothing asked for
