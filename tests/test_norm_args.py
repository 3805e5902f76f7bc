"""Calls of the norms that are refused, before anything is launched (host only)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mintext_amd import _lib as L
from mintext_amd.kernels import layer_norm, rms_norm


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


F32 = torch.float32


@pytest.mark.parametrize("norm", [layer_norm, rms_norm])
@pytest.mark.parametrize("args, kwargs, error", [
    ((z(4, 8), z(9)), {}, ValueError),                                     # widths differ
    ((z(4, 8), z(1, 8)), {}, ValueError),
    ((z(()), z(1)), {}, ValueError),                                       # no dimension
    ((z(4, 0), z(0)), {}, ValueError),                                     # no width
    ((z(4, 16385), z(16385)), {}, ValueError),                             # wider than the registers
    ((z(4, 8), z(8)), dict(residual=z(8)), ValueError),                    # broadcast by the caller, not here
    ((z(4, 8), z(8)), dict(eps=-1e-6), ValueError),
    ((z(4, 8), z(8)), dict(eps=float("nan")), ValueError),
    ((z(4, 8), z(8)), dict(residual=z(4, 8, dtype=F32)), TypeError),
    ((z(4, 8, dtype=F32), z(8)), {}, TypeError),                           # a bfloat16 weight beside float32 rows
    ((z(4, 8, dtype=torch.float16), z(8, dtype=torch.float16)), {}, TypeError),
    ((z(4, 8), z(8)), {}, RuntimeError),                                   # no device
])
def test_refusals(norm, args, kwargs, error):
    with pytest.raises(error):
        norm(*args, **kwargs)


def test_bias_refusals():
    with pytest.raises(ValueError):
        layer_norm(z(4, 8), z(8), z(7))
    with pytest.raises(TypeError):
        layer_norm(z(4, 8), z(8), z(8, dtype=F32))


def test_entry_points_refuse():
    lib = L.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    d, P, n = ctypes.addressof(buf) // 16 * 16 + 16, None, 1 << 15
    size = lib.mtx_norm_bwd_workspace_size
    assert size(4, 8) > 0 and size(0, 8) > 0 and size(-1, 8) < 0 and size(4, 0) < 0 and size(4, 16385) < 0
    fwd = lambda x=d, r=P, w=d, b=P, dt=1, wt=1, rms=0, T=4, D=8, eps=1e-5, y=d, h=P, m=d, s=d: lib.mtx_norm(
        x, r, w, b, dt, wt, rms, T, D, eps, y, h, m, s, P)
    assert fwd(dt=2) == L.MTX_ERR_ARG and fwd(dt=0, wt=1) == L.MTX_ERR_ARG        # dtypes
    assert fwd(T=-1) == L.MTX_ERR_ARG and fwd(D=0) == L.MTX_ERR_ARG
    assert fwd(D=16385) == L.MTX_ERR_UNSUPPORTED and fwd(T=1 << 31) == L.MTX_ERR_UNSUPPORTED
    assert fwd(eps=-1.0) == L.MTX_ERR_ARG and fwd(rms=1, b=d) == L.MTX_ERR_ARG
    assert fwd(x=P) == L.MTX_ERR_ARG and fwd(w=P) == L.MTX_ERR_ARG and fwd(y=P) == L.MTX_ERR_ARG
    assert fwd(r=d) == L.MTX_ERR_ARG                                              # nowhere to write the sum
    assert fwd(m=P) == L.MTX_ERR_ARG                                              # rstd without mean
    assert fwd(T=0) == L.MTX_OK
    bwd = lambda dy=d, dh=P, h=d, w=d, m=d, s=d, dt=1, wt=1, rms=0, T=4, D=8, dx=d, dw=d, db=d, ws=d, size=n: lib.mtx_norm_bwd(
        dy, dh, h, w, m, s, dt, wt, rms, T, D, dx, dw, db, ws, size, P)
    assert bwd(dt=2) == L.MTX_ERR_ARG and bwd(rms=1) == L.MTX_ERR_ARG             # a bias of an RMS norm
    assert bwd(dw=P) == L.MTX_ERR_ARG                                             # dbias without dweight
    assert bwd(dx=P, dw=P, db=P) == L.MTX_OK                                      # nothing asked for
    for missing in ("dy", "h", "w", "m", "s"):
        assert bwd(**{missing: P}) == L.MTX_ERR_ARG, missing
    assert bwd(ws=P) == L.MTX_ERR_WORKSPACE and bwd(size=8) == L.MTX_ERR_WORKSPACE
    assert bwd(D=16385) == L.MTX_ERR_UNSUPPORTED
