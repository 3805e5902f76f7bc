"""Layer norm and RMS norm of rows, with the residual's addition in front, differentiable.

``rms_norm`` is the reference's ``RMSNorm`` (mintext/modules/norm.py:10), the norm in front of every block and of the
head; ``layer_norm`` is its form with mean and bias.  With ``residual`` one pass computes the new residual stream
``h = x + residual`` and its norm.  One HIP kernel reads each tensor once; the backward is one pass over ``h`` and the
gradients and a sum of its workgroups' shares of the weight's and bias's gradients, in a fixed order.
"""
from __future__ import annotations

import torch

from .. import _lib as L

MAX_WIDTH = 16384


def _check(name, x, weight, bias, residual, eps):
    xs = x.shape
    if len(xs) < 1 or weight.shape != (xs[-1],):
        raise ValueError(f"{name} takes x [..., D] and weight [D], got {tuple(xs)} and {tuple(weight.shape)}")
    if not 0 < xs[-1] <= MAX_WIDTH:
        raise ValueError(f"{name} takes widths of 1 to {MAX_WIDTH}, got {xs[-1]}")
    if bias is not None and bias.shape != weight.shape:
        raise ValueError(f"bias must be [{xs[-1]}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != xs:
        raise ValueError(f"residual must have x's shape {tuple(xs)}, got {tuple(residual.shape)}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float32:
        raise TypeError(f"{name} takes float32 or bfloat16 tensors, got {dt}")
    if residual is not None and residual.dtype is not dt:
        raise TypeError(f"residual must have x's dtype {dt}, got {residual.dtype}")
    wt = weight.dtype
    if (wt is not dt and wt is not torch.float32) or (bias is not None and bias.dtype is not wt):
        raise TypeError(f"weight and bias must share one dtype, {dt} as x or float32")


def _forward(x, residual, weight, bias, rms, eps, keep):
    """y, h, what the backward needs of each row (1 / sqrt(variance + eps), behind it the means), and its sizes and type codes."""
    dev = L.require_device(x, residual, weight, bias)
    D = int(x.shape[-1])  # numbers, also where a jit trace has sizes of its own: it calls the Function again for other tensors
    T = int(x.numel() // D)
    x, weight = x.contiguous(), weight.contiguous()
    y = torch.empty_like(x)
    r = b = h = m = s = stats = None  # the letters: addresses
    if residual is not None:
        residual = residual.contiguous()
        hidden = torch.empty_like(x)
        r, h = residual.data_ptr(), hidden.data_ptr()
    else:
        hidden = x
    if bias is not None:
        bias = bias.contiguous()
        b = bias.data_ptr()
    if keep:
        stats = torch.empty(T if rms else 2 * T, dtype=torch.float32, device=dev)
        s = stats.data_ptr()
        if not rms:
            m = s + 4 * T
    how = (L.dtype_code(x.dtype), L.dtype_code(weight.dtype), rms, T, D)
    with L.on_device(dev):
        L.call("mtx_norm", x.data_ptr(), r, weight.data_ptr(), b, *how, eps, y.data_ptr(), h, m, s, L.stream(dev))
    return y, hidden, stats, how


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, rms, eps):
        y, h, stats, how = _forward(x, residual, weight, bias, rms, eps, True)
        ctx.save_for_backward(h, weight, stats)
        # worked out here: the backward runs in a thread of its own, where each step may cost two to three times as much
        ctx.how = how, L.query("mtx_norm_bwd_workspace_size", *how[3:])
        ctx.set_materialize_grads(False)
        return (y, h) if residual is not None else y

    @staticmethod
    @L.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, stats = ctx.saved_tensors
        need_x, need_r, need_w, need_b, _, _ = ctx.needs_input_grad
        if dy is None:  # the sum alone is used
            return (dh if need_x else None, dh if need_r else None, None, None, None, None)
        how, nbytes = ctx.how
        rms, T = how[2:4]
        dev = L.require_device(dy, dh, h)
        dy, weight = dy.contiguous(), weight.contiguous()
        dx = dw = db = None
        dhp = dxp = dwp = dbp = wsp = None
        if dh is not None:
            dh = dh.contiguous()
            dhp = dh.data_ptr()
        if need_x or need_r:
            dx = torch.empty_like(h)
            dxp = dx.data_ptr()
        if need_w or need_b:
            dw = torch.empty_like(weight)
            ws = L.workspace(nbytes, dev)
            dwp, wsp = dw.data_ptr(), ws.data_ptr()
        if need_b:
            db = torch.empty_like(weight)
            dbp = db.data_ptr()
        rstd = stats.data_ptr()
        with L.on_device(dev):
            L.call("mtx_norm_bwd", dy.data_ptr(), dhp, h.data_ptr(), weight.data_ptr(), None if rms else rstd + 4 * T, rstd, *how,
                   dxp, dwp, dbp, wsp, nbytes, L.stream(dev))
        return dx if need_x else None, dx if need_r else None, dw if need_w else None, db, None, None


def _norm(name, x, weight, bias, rms, eps, residual):
    eps = float(eps)
    _check(name, x, weight, bias, residual, eps)
    if L.plain_forward(x, weight, bias, residual):
        y, h, _, _ = _forward(x, residual, weight, bias, rms, eps, False)
        return y if residual is None else (y, h)
    return _Norm.apply(x, residual, weight, bias, rms, eps)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, eps: float = 1e-5,
               residual: torch.Tensor | None = None):
    """``(h - mean(h)) / sqrt(var(h) + eps) * weight + bias`` over the last dimension, ``h = x + residual``.

    Args:
        x: [..., D], float32 or bfloat16, D up to 16384.
        weight: [D], in x's dtype or float32.
        bias: [D] in the weight's dtype, or None.
        residual: x's shape and dtype, or None.

    Returns:
        y in x's shape and dtype; with ``residual`` (y, h), where ``h`` is the sum rounded to x's dtype, of which the
        norm is taken.  Statistics are in float32.  Differentiable (once) in all four tensors.
    """
    return _norm("layer_norm", x, weight, bias, False, eps, residual)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor | None = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension (mintext/modules/norm.py:10), ``h = x + residual``.

    Arguments, results and gradients as ``layer_norm``'s, without a bias.
    """
    return _norm("rms_norm", x, weight, None, True, eps, residual)
