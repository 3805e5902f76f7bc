"""Dense product with its epilogue: ``act(x @ weight + bias) + residual``, differentiable.

The dense counterpart of ``grouped_matmul``, for the projections and MLPs around the experts (the reference's
``Linear`` and ``MLP``, mintext/modules/linear.py:123-147, 164-228): one HIP kernel applies bias, activation and
residual to the float32 sums, rounded once.  Training also writes ``z = x @ weight + bias``, in the operands' dtype,
when there is an activation; its backward is one pass over the gradient and ``z`` (``dz = dy * act'(z)`` and the
bias gradient) and the two products ``dz @ weight^T`` and ``x^T @ dz``.  ``dz`` is rounded to the operands' dtype for the
products (the bias gradient sums it before), so that bfloat16 gradients behind an activation end 2.4e-3 off (2-norm)
where the rounding of the result alone is 1.7e-3.  The gradients are deterministic.

bfloat16 runs on the 16-bit matrix cores where K and N are multiples of 8 and the tensors lie on 16-byte boundaries;
otherwise its products run in float32, at less than a tenth of the rate where they are large (4096 x 2048 x 50257 takes
12.5 ms, with 50264 columns 0.78): such widths are worth padding.  float32 runs at up to 116 TFLOP/s, level with a
library's products and separate passes.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib as L

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}  # MTX_ACT_*


def _check(x, weight, bias, activation, residual):
    """The activation's code; a serving call spends as long on the host as on the GPU, hence no loops."""
    act = ACTIVATIONS.get(activation, -1)
    if act < 0:
        raise ValueError(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)} or None, got {activation!r}")
    xs, ws = x.shape, weight.shape
    if len(xs) < 1 or len(ws) != 2 or xs[-1] != ws[0]:
        raise ValueError(f"linear takes x [..., K] and weight [K, N], got {tuple(xs)} and {tuple(ws)}")
    K, N = ws
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*xs[:-1], N):
        raise ValueError(f"residual must have the output's shape {(*xs[:-1], N)}, got {tuple(residual.shape)}")
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float32:
        raise TypeError(f"linear takes float32 or bfloat16 operands, got {dt}")
    if (weight.dtype is not dt or (bias is not None and bias.dtype is not dt)
            or (residual is not None and residual.dtype is not dt)):
        raise TypeError(f"linear operands must share one dtype, {dt} as x")
    return act


def _sizes(x, weight):
    K, N = weight.shape
    return (x.numel() // K if K else math.prod(x.shape[:-1])), K, N


def _forward(x, weight, bias, residual, act, keep):
    dev = L.require_device(x, weight, bias, residual)
    M, K, N = _sizes(x, weight)
    x, weight = x.contiguous(), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=dev)
    pre = torch.empty((M, N), dtype=x.dtype, device=dev) if keep and act else None
    ws = L.workspace(L.query("mtx_linear_workspace_size", M, K, N), dev)
    with L.on_device(dev):
        L.call("mtx_linear", x.data_ptr(), weight.data_ptr(), L.ptr(bias), L.ptr(residual), L.dtype_code(x.dtype), M, K, N,
               act, out.data_ptr(), L.ptr(pre), ws.data_ptr(), ws.numel(), L.stream(dev))
    return out, pre


class _Linear(torch.autograd.Function):
    # The sizes are taken in here: a jit trace calls this again for other tensors, with its first call's other arguments.
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        out, pre = _forward(x, weight, bias, residual, act, True)
        ctx.save_for_backward(x, weight, pre)
        ctx.act = act
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dev = L.require_device(x, weight, dy)
        x, weight, dy = x.contiguous(), weight.contiguous(), dy.contiguous()
        (M, K, N), act = _sizes(x, weight), ctx.act
        dz = torch.empty((M, N), dtype=x.dtype, device=dev) if act and (need_x or need_w or need_b) else None
        dx = torch.empty_like(x) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty(N, dtype=x.dtype, device=dev) if need_b else None
        ws = L.workspace(L.query("mtx_linear_workspace_size", M, K, N), dev)
        with L.on_device(dev):
            L.call("mtx_linear_bwd", L.ptr(dy), L.ptr(x), L.ptr(weight), L.ptr(pre), L.dtype_code(x.dtype), M, K, N, act,
                   L.ptr(dz), L.ptr(dx), L.ptr(dw), L.ptr(db), L.ptr(ws), ws.numel(), L.stream(dev))
        return dx, dw, db, dy if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight + bias) + residual`` as one kernel (the products of mintext/modules/linear.py:123-147, 164-228).

    Args:
        x: [..., K], float32 or bfloat16.
        weight: [K, N] in x's dtype (the layout of ``grouped_matmul``'s weights, one group).
        bias: [N] or None.
        activation: None, "relu", "silu", "gelu" (erf) or "gelu_tanh".
        residual: [..., N] or None, added after the activation.

    Returns:
        [..., N] in x's dtype.  Differentiable (once) in all four tensors.
    """
    act = _check(x, weight, bias, activation, residual)
    if L.plain_forward(x, weight, bias, residual):
        return _forward(x, weight, bias, residual, act, False)[0]
    return _Linear.apply(x, weight, bias, residual, act)
