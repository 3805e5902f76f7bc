"""Calls of newton_schulz and muon_update that are refused, and their schedules (host only)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from mintext_amd import _lib as L
from mintext_amd.kernels import muon_update, newton_schulz
from mintext_amd.kernels.muon import COEFFICIENTS, _schedule


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("x, kwargs, error", [
    (z(8), {}, ValueError),
    (z(4, 8, dtype=torch.float16), {}, TypeError),
    (z(4, 8), dict(steps=0), ValueError),
    (z(4, 8), dict(steps=65), ValueError),
    (z(4, 8), dict(steps=2.0), ValueError),
    (z(4, 8), dict(eps=0.0), ValueError),
    (z(4, 8), dict(precision="bf16"), ValueError),
    (z(4, 8), dict(coefficients=(1.0, 2.0)), ValueError),
    (z(4, 8), dict(coefficients=((1.5, -0.5, 0.0),) * 4), ValueError),       # four triples for five steps
    (z(4, 8), dict(coefficients=(1.5, float("nan"), 0.0)), ValueError),
    (z(4, 8), dict(coefficients=(30.0, 30.0, 30.0)), ValueError),            # the steps diverge
    (z(4, 8).requires_grad_(True), {}, RuntimeError),
    (z(4, 8), {}, RuntimeError),                                             # no device
])
def test_newton_schulz_refuses(x, kwargs, error):
    with pytest.raises(error):
        newton_schulz(x, **kwargs)


P, G, M = z(3, 4, 8), z(3, 4, 8), z(3, 4, 8)


@pytest.mark.parametrize("args, kwargs, error", [
    ((P, z(3, 8, 4), M), dict(lr=0.1), ValueError),
    ((P, G, z(3, 4, 7)), dict(lr=0.1), ValueError),
    ((P, G, z(3, 4, 8, dtype=torch.bfloat16)), dict(lr=0.1), TypeError),     # momentum is float32
    ((P, G, M), dict(lr=torch.zeros(2)), TypeError),
    ((P, G, M), dict(lr=torch.zeros(1, dtype=torch.float64)), TypeError),
    ((P, G, M), dict(lr=0.1, scale="fan"), ValueError),
    ((P, G, P), dict(lr=0.1), ValueError),                                   # one tensor twice
    ((P, P, M), dict(lr=0.1), ValueError),
    ((z(3, 8, 4).mT, G, M), dict(lr=0.1), ValueError),                       # rows of strided elements, in place
    ((z(1, 4, 8).expand(3, 4, 8), G, M), dict(lr=0.1), ValueError),          # the same memory three times
    ((P, G, z(3, 1, 8).expand(3, 4, 8)), dict(lr=0.1), ValueError),
    ((z(4, 5, 4, 8).transpose(0, 1), z(5, 4, 4, 8), z(5, 4, 4, 8)), dict(lr=0.1), ValueError),  # not one batch
    ((P, G, M), dict(lr=0.1), RuntimeError),                                 # no device
])
def test_muon_update_refuses(args, kwargs, error):
    with pytest.raises(error):
        muon_update(*args, **kwargs)


@pytest.mark.parametrize("group", [1, 2, 3])
@pytest.mark.parametrize("steps", range(1, 10))
def test_schedule(steps, group):
    s = list(_schedule(steps, COEFFICIENTS, group))
    rows = [s[9 * i:9 * i + 9] for i in range(steps)]
    ends = [r[8] for r in rows]
    assert ends[-1] == 1.0
    size, sizes = 0, []
    for e in ends:
        size += 1
        if e:
            sizes.append(size)
            size = 0
    assert sum(sizes) == steps and max(sizes) <= group and sizes == sorted(sizes, reverse=True)
    first = True
    for r in rows:
        assert all(math.log2(v).is_integer() for v in r[3:8])
        assert not first or r[6] == r[4]  # P is Q at a group's first step
        first = bool(r[8])
    # every entry of every matrix stays in f16: its bound times its scale
    sv = [k / 1000 for k in range(1001)]
    p = [1.0] * 1001
    for r in rows:
        a, b, c, sa, sq, st, sp, sx, end = r
        q = [a + b * t * t + c * t ** 4 for t in sv]
        p = [u * v for u, v in zip(p, q)]
        assert max(t * t for t in sv) * sa < 65504 and max(map(abs, q)) * sq < 65504
        assert max(abs(v) * t * t for v, t in zip(q, sv)) * st < 65504 and max(map(abs, p)) * sp < 65504
        sv = [abs(v) * t for v, t in zip(q, sv)]
        assert max(sv) * sx < 65504
        if end:
            p = [1.0] * 1001


def test_entry_points_refuse():
    lib = L.lib()
    buf = ctypes.create_string_buffer(4096)
    d, N_ = ctypes.addressof(buf), None
    sched = _schedule(5, COEFFICIENTS, 3)
    size = lib.mtx_newton_schulz_workspace_size
    assert size(4, 64, 32, 1) > 0 and size(4, 64, 32, 2) > size(4, 64, 32, 1)
    assert size(4, 64, 32, 3) < 0 and size(-1, 64, 32, 1) < 0 and size(1, 1 << 16, 1 << 16, 1) < 0
    assert size(0, 64, 32, 1) == 0

    def call(dtype=0, E=2, M=8, N=8, row=8, sched=sched, steps=5, eps=1e-7, planes=1, x=d, out=d, ws=d, n=1 << 40):
        return lib.mtx_newton_schulz(x, dtype, E, M, N, M * row, row, sched, steps, eps, planes, out, M * N, N, ws, n, N_)

    assert call(dtype=2) == L.MTX_ERR_ARG
    assert call(row=7) == L.MTX_ERR_ARG          # rows that overlap
    assert call(steps=0) == L.MTX_ERR_ARG and call(sched=N_) == L.MTX_ERR_ARG
    assert call(eps=0.0) == L.MTX_ERR_ARG and call(planes=0) == L.MTX_ERR_ARG
    assert call(x=N_) == L.MTX_ERR_ARG and call(out=N_) == L.MTX_ERR_ARG
    assert call(n=64) == L.MTX_ERR_WORKSPACE and call(ws=N_) == L.MTX_ERR_WORKSPACE
    assert call(M=1 << 21) == L.MTX_ERR_UNSUPPORTED
    bad = (ctypes.c_float * 45)(*sched)
    bad[4] = 0.0
    assert call(sched=bad) == L.MTX_ERR_ARG
    assert call(E=0) == L.MTX_OK
    step = lambda pt, gt, m: lib.mtx_muon_update(d, pt, 64, 8, d, gt, 64, 8, m, 64, 8, 2, 8, 8, 0.9, 1, 0.1, N_, 0.0, 1.0,
                                                 sched, 5, 1e-7, 1, d, 1 << 40, N_)
    assert step(2, 0, d) == L.MTX_ERR_ARG and step(0, 2, d) == L.MTX_ERR_ARG and step(0, 0, N_) == L.MTX_ERR_ARG
