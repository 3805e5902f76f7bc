"""Calls of the head's losses that are refused, before anything is launched (host only)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mintext_amd import _lib as L
from mintext_amd.kernels import linear_cross_entropy, linear_distillation

BF, F32 = torch.bfloat16, torch.float32


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def i(*shape, dtype=torch.int64):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args, kwargs, error", [
    ((z(4, 8), z(9, 16), i(4)), {}, ValueError),                             # widths differ
    ((z(4, 8), z(2, 8, 16), i(4)), {}, ValueError),                          # a stack of weights
    ((z(4, 0), z(0, 16), i(4)), {}, ValueError),
    ((z(4, 8), z(8, 0), i(4)), {}, ValueError),                              # no vocabulary
    ((z(4, 8), z(8, 16), i(5)), {}, ValueError),
    ((z(4, 8), z(8, 16), i(4, 1)), {}, ValueError),
    ((z(4, 8), z(8, 16), i(4)), dict(reduction="batchmean"), ValueError),
    ((z(4, 8), z(8, 16), i(4)), dict(z_loss=-1e-4), ValueError),
    ((z(4, 8), z(8, 16), i(4)), dict(z_loss=float("nan")), ValueError),
    ((z(4, 8), z(8, 16), i(4)), dict(ignore_index=1 << 63), ValueError),
    ((z(4, 8), z(8, 16, dtype=F32), i(4)), {}, TypeError),                   # mixed types
    ((z(4, 8, dtype=torch.float16), z(8, 16, dtype=torch.float16), i(4)), {}, TypeError),
    ((z(4, 8), z(8, 16), z(4, dtype=F32)), {}, TypeError),                   # targets that are no integers
    ((z(4, 8), z(8, 16), i(4, dtype=torch.int16)), {}, TypeError),
    ((z(4, 8), z(8, 16), i(4)), {}, RuntimeError),                           # no device
])
def test_cross_entropy_refusals(args, kwargs, error):
    with pytest.raises(error):
        linear_cross_entropy(*args, **kwargs)


T3, I3 = z(4, 3, dtype=F32), i(4, 3)


@pytest.mark.parametrize("args, kwargs, error", [
    ((z(4, 8), z(9, 16), I3, T3), {}, ValueError),
    ((z(4, 8), z(8, 16), i(4), z(4, dtype=F32)), {}, ValueError),            # no dimension of entries
    ((z(4, 8), z(8, 16), I3, z(4, 2, dtype=F32)), {}, ValueError),
    ((z(4, 8), z(8, 16), i(5, 3), z(5, 3, dtype=F32)), {}, ValueError),
    ((z(4, 8), z(8, 16), i(4, 0), z(4, 0, dtype=F32)), {}, ValueError),
    ((z(4, 8), z(8, 16), i(4, 1025), z(4, 1025, dtype=F32)), {}, ValueError),
    ((z(4, 8), z(8, 16), I3, T3), dict(temperature=0.0), ValueError),
    ((z(4, 8), z(8, 16), I3, T3), dict(temperature=float("nan")), ValueError),
    ((z(4, 8), z(8, 16), I3, T3), dict(temperature=float("inf")), ValueError),
    ((z(4, 8), z(8, 16), I3, T3), dict(reduction="max"), ValueError),
    ((z(4, 8), z(8, 16), T3, T3), {}, TypeError),
    ((z(4, 8), z(8, 16), I3, T3.double()), {}, TypeError),
    ((z(4, 8), z(8, 16), I3, T3), {}, RuntimeError),                         # no device
])
def test_distillation_refusals(args, kwargs, error):
    with pytest.raises(error):
        linear_distillation(*args, **kwargs)


def test_workspace_sizes():
    lib = L.lib()
    size, held = lib.mtx_head_loss_workspace_size, lib.mtx_distillation_entries_size
    assert size(L.MTX_BF16, 16, 8, 100, 0, 0) > 0 and size(L.MTX_F32, 0, 8, 100, 1, 1) > 0
    for bad in ((2, 16, 8, 100, 0, 0), (1, -1, 8, 100, 0, 0), (1, 16, 0, 100, 0, 0), (1, 16, 8, 0, 0, 0), (1, 16, 8, 100, 2, 0),
                (1, 1 << 23, 8, 100, 0, 0), (1, 16, 8, 1 << 23, 0, 0)):
        assert size(*bad) < 0, bad
    assert held(4, 100, 3) > 0 and held(0, 100, 3) > 0
    assert held(4, 100, 0) < 0 and held(4, 100, 1025) < 0 and held(-1, 100, 3) < 0
    # the gradient's workspace does not grow with the vocabulary beyond a piece's: 1 GiB of dz, dx in 32 bits, some more
    dx = 65536 * 4096 * 4
    for V in (65536, 262144, 1048576):
        assert size(L.MTX_BF16, 65536, 4096, V, 0, 1) <= (1 << 30) + dx + (1 << 24)
    # and the forward's keeps 8 bytes for 64 logits at most
    assert size(L.MTX_BF16, 8192, 4096, 131072, 0, 0) <= 8192 * 131072 // 8


def test_entry_points_refuse():
    lib = L.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    d, P = ctypes.addressof(buf) // 16 * 16 + 16, None
    big = 1 << 40
    ce = lambda x=d, w=d, y=d, dt=1, T=4, D=8, V=16, order=0, zl=0.0, loss=d, lse=d, st=d, total=d, count=d, ch=d, ws=d, n=big: \
        lib.mtx_linear_cross_entropy(x, w, y, 1, dt, T, D, V, order, -100, zl, 1, loss, lse, st, total, count, ch, ws, n, P)
    assert ce(dt=2) == ce(order=2) == ce(T=-1) == ce(D=0) == ce(V=0) == ce(zl=-1.0) == ce(zl=float("inf")) == L.MTX_ERR_ARG
    assert ce(T=1 << 23) == ce(V=1 << 23) == L.MTX_ERR_UNSUPPORTED
    assert ce(total=P) == ce(count=P) == L.MTX_ERR_ARG                           # one without the other
    for missing in ("x", "w", "y", "loss", "lse", "st", "ch"):
        assert ce(**{missing: P}) == L.MTX_ERR_ARG, missing
    assert ce(x=d + 2) == ce(w=d + 8) == L.MTX_ERR_ARG                           # off a 16-byte boundary
    assert ce(ws=P) == ce(n=16) == ce(ws=d + 4) == L.MTX_ERR_WORKSPACE
    ceb = lambda g=d, x=d, w=d, y=d, lse=d, st=d, ch=d, dt=1, T=4, V=16, dx=d, dw=d, ws=d, n=big: lib.mtx_linear_cross_entropy_bwd(
        g, P, x, w, y, 1, lse, st, ch, dt, T, 8, V, 0, 0.0, dx, dw, ws, n, P)
    assert ceb(dt=2) == L.MTX_ERR_ARG and ceb(V=1 << 23) == L.MTX_ERR_UNSUPPORTED
    assert ceb(dx=P, dw=P) == ceb(T=0) == L.MTX_OK                               # nothing to do
    for missing in ("g", "x", "w", "y", "lse", "st", "ch"):
        assert ceb(**{missing: P}) == L.MTX_ERR_ARG, missing
    assert ceb(ws=P) == ceb(n=16) == L.MTX_ERR_WORKSPACE
    kd = lambda x=d, w=d, i=d, t=d, tt=0, dt=1, T=4, K=3, tau=1.0, loss=d, lse=d, st=d, ch=d, e=d, en=big, ws=d, n=big: \
        lib.mtx_linear_distillation(x, w, i, 0, t, tt, dt, T, 8, 16, K, 0, tau, 1, loss, lse, st, d, d, ch, e, en, ws, n, P)
    assert kd(dt=2) == kd(tt=2) == kd(K=0) == kd(tau=0.0) == kd(tau=float("nan")) == kd(tau=float("inf")) == L.MTX_ERR_ARG
    assert kd(K=1025) == L.MTX_ERR_UNSUPPORTED
    for missing in ("x", "w", "i", "t", "loss", "lse", "st", "ch", "e"):
        assert kd(**{missing: P}) == L.MTX_ERR_ARG, missing
    assert kd(en=16) == kd(e=d + 4) == kd(ws=P) == kd(n=16) == L.MTX_ERR_WORKSPACE
    kdb = lambda g=d, x=d, w=d, e=d, en=big, lse=d, st=d, ch=d, T=4, K=3, tau=1.0, dx=d, dw=d, ws=d, n=big: \
        lib.mtx_linear_distillation_bwd(g, P, x, w, e, en, lse, st, ch, 1, T, 8, 16, K, 0, tau, dx, dw, ws, n, P)
    assert kdb(K=0) == kdb(tau=-1.0) == L.MTX_ERR_ARG and kdb(K=1025) == L.MTX_ERR_UNSUPPORTED
    assert kdb(T=0) == kdb(dx=P, dw=P) == L.MTX_OK
    for missing in ("g", "x", "w", "e", "lse", "st", "ch"):
        assert kdb(**{missing: P}) == L.MTX_ERR_ARG, missing
    assert kdb(en=16) == kdb(ws=P) == kdb(n=16) == L.MTX_ERR_WORKSPACE
