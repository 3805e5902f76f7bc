"""Losses of a vocabulary-sized head without its logits in memory, differentiable.

``linear_cross_entropy`` is the reference's vocabulary-tiled loss with its z-loss (mintext/trainer.py:197-241);
``linear_distillation`` is the same against a teacher's top logits.  Both take the head's input and its weight: one kernel
makes the logits tile by tile on the matrix cores and leaves each tile's maxima, sums and the logits that the loss
names; the [T, V] logits are not stored, in neither direction.  The backward makes them again in pieces of the
vocabulary whose gradient takes 1 GiB at most (or 320 columns of it, where the tokens are so many that those take more), and runs
the two products of each piece; over the pieces the gradient of ``x`` is summed in float32.  The gradient of the logits is rounded
to the operands' type for the products (bfloat16: as in ``linear``'s backward, the results end 2.4e-3 off where their own rounding
is 1.7e-3; up to 64 tokens keep what that rounding took as well, and end at their own).  Every sum has a fixed order.

The weight is [D, V] as it lies in memory, or an embedding table [V, D] passed as ``table.t()``: both are read in place, and
the weight's gradient has the weight's strides.  In bfloat16 a vocabulary (or, for a table, a width) that is no multiple of 8
costs a padded copy of the weight, piece by piece, in each direction.

In float32 a loss with its gradients takes 1.4 to 1.7 times as long as with the logits in memory where both the tokens (more than 64)
and the vocabulary are many: four products in tiles that reach half to three quarters of a library's rate, for three.  What it
saves there is memory.
"""
from __future__ import annotations

import math

import torch

from .. import _lib as L

REDUCTIONS = ("mean", "sum", "none")
MAX_ENTRIES = 1024


def _check(name, x, weight, reduction):
    xs, ws = x.shape, weight.shape
    if len(xs) < 1 or len(ws) != 2 or xs[-1] != ws[0]:
        raise ValueError(f"{name} takes x [..., D] and weight [D, V], got {tuple(xs)} and {tuple(ws)}")
    if ws[0] == 0 or ws[1] == 0:
        raise ValueError(f"{name} needs a width and a vocabulary, got weight {tuple(ws)}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {REDUCTIONS}, got {reduction!r}")
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float32:
        raise TypeError(f"{name} takes float32 or bfloat16 operands, got {dt}")
    if weight.dtype is not dt:
        raise TypeError(f"x and weight must share one dtype, got {dt} and {weight.dtype}")


def _dense(x, weight):
    """x, and the weight with its order in memory: as it is where it is dense in one and on a 16-byte boundary."""
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    order = L.MTX_HEAD_DV
    if not weight.is_contiguous():
        if weight.t().is_contiguous():
            order = L.MTX_HEAD_VD
        else:
            weight = weight.contiguous()
    if weight.data_ptr() % 16:
        weight = weight.clone()  # strides are kept
    return x, weight, order


def _index64(name, t):
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    return int(t.dtype is torch.int64)


class _Loss:
    """One of the two losses: what it calls, and what its backward needs beside x and the weight."""

    def __init__(self, reduction, z_loss=0.0, ignore_index=0, temperature=1.0):
        self.reduction, self.z_loss, self.ignore_index, self.temperature = reduction, z_loss, ignore_index, temperature

    @staticmethod
    def rows(buffer, T, K):
        """Addresses in the float32 buffer of maxima and sums [T, 2], state [T], the named logits [T, K], the count, the losses [T].
        (Numbers, also where a jit trace has sizes of its own: it calls the Function again for other tensors.)"""
        at = buffer.data_ptr()
        return at, at + 8 * T, at + 12 * T, at + 4 * (3 + K) * T, at + 4 * (3 + K) * T + 4

    def forward(self, x, weight, classes, teacher):
        dev = L.require_device(x, weight, classes, teacher)
        D, V = weight.shape
        T, K = int(x.numel() // D), 1 if teacher is None else int(classes.shape[-1])
        x, weight, order = _dense(x, weight)
        classes = classes.contiguous()
        dt, wide = L.dtype_code(x.dtype), _index64("classes", classes)
        # the result is a tensor of its own, which a caller may change in place
        one = self.reduction != "none"
        out = torch.empty(() if one else x.shape[:-1], dtype=torch.float32, device=dev)
        buffer = torch.empty((3 + K + one) * T + 1, dtype=torch.float32, device=dev)
        stats, state, chosen, count, loss = self.rows(buffer, T, K)
        total = out.data_ptr() if one else None
        if not one:
            count, loss = None, out.data_ptr()
        mean = int(self.reduction == "mean")
        ws = L.workspace(L.query("mtx_head_loss_workspace_size", dt, T, D, V, order, 0), dev)
        kept = classes
        with L.on_device(dev):
            if teacher is None:
                L.call("mtx_linear_cross_entropy", x.data_ptr(), weight.data_ptr(), classes.data_ptr(), wide, dt, T, D, V, order,
                       self.ignore_index, self.z_loss, mean, loss, stats, state, total, count, chosen, ws.data_ptr(), ws.numel(),
                       L.stream(dev))
            else:
                teacher = teacher.contiguous()
                kept = L.workspace(L.query("mtx_distillation_entries_size", T, V, K), dev)
                L.call("mtx_linear_distillation", x.data_ptr(), weight.data_ptr(), classes.data_ptr(), wide, teacher.data_ptr(),
                       L.dtype_code(teacher.dtype), dt, T, D, V, K, order, self.temperature, mean, loss, stats, state, total, count,
                       chosen, kept.data_ptr(), kept.numel(), ws.data_ptr(), ws.numel(), L.stream(dev))
        return out, (x, weight, kept, buffer)

    def backward(self, g, x, weight, kept, buffer, K, need_x, need_w):
        dev = L.require_device(g, x, weight)
        D, V = weight.shape
        T = int(x.numel() // D)
        order = L.MTX_HEAD_DV if weight.is_contiguous() else L.MTX_HEAD_VD
        g = g.contiguous()
        stats, state, chosen, count, _ = self.rows(buffer, T, K or 1)
        if self.reduction == "none":
            count = None
        dt = L.dtype_code(x.dtype)
        dx = torch.empty_like(x) if need_x else None
        dw = (torch.empty_like(weight) if T else torch.zeros_like(weight)) if need_w else None  # with the weight's strides
        ws = L.workspace(L.query("mtx_head_loss_workspace_size", dt, T, D, V, order, 1), dev)
        with L.on_device(dev):
            if K is None:
                L.call("mtx_linear_cross_entropy_bwd", g.data_ptr(), count, x.data_ptr(), weight.data_ptr(), kept.data_ptr(),
                       _index64("classes", kept), stats, state, chosen, dt, T, D, V, order, self.z_loss, L.ptr(dx), L.ptr(dw),
                       ws.data_ptr(), ws.numel(), L.stream(dev))
            else:
                L.call("mtx_linear_distillation_bwd", g.data_ptr(), count, x.data_ptr(), weight.data_ptr(), kept.data_ptr(),
                       kept.numel(), stats, state, chosen, dt, T, D, V, K, order, self.temperature, L.ptr(dx), L.ptr(dw),
                       ws.data_ptr(), ws.numel(), L.stream(dev))
        return dx, dw


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, classes, teacher, how):
        out, saved = how.forward(x, weight, classes, teacher)
        ctx.save_for_backward(*saved)
        ctx.how, ctx.K = how, None if teacher is None else int(classes.shape[-1])
        return out

    @staticmethod
    @L.once_differentiable
    def backward(ctx, g):
        need_x, need_w = ctx.needs_input_grad[:2]
        return (*ctx.how.backward(g, *ctx.saved_tensors, ctx.K, need_x, need_w), None, None, None)


def _loss(x, weight, classes, teacher, how):
    if L.plain_forward(x, weight):
        return how.forward(x, weight, classes, teacher)[0]
    return _HeadLoss.apply(x, weight, classes, teacher, how)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         z_loss: float = 0.0, reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of ``x @ weight`` against ``targets``, plus ``z_loss * logsumexp^2`` (trainer.py:197-241).

    Args:
        x: [..., D], float32 or bfloat16.
        weight: [D, V] in x's dtype, dense in either order (``table.t()`` of an embedding table [V, D]).
        targets: [...] int32 or int64; tokens whose target is ``ignore_index`` have no loss and no gradient.  A target
            outside [0, V) that is not ``ignore_index`` makes its token's loss and gradient NaN.
        z_loss: factor of the squared logarithm of the sum of exponentials, not negative.
        reduction: "mean" over the tokens that are not ignored (0 if all are), "sum", or "none".

    Returns:
        The loss, float32: a scalar, or [...] for "none".  Differentiable (once) in x and weight.  An ignored token's x has to
        be finite for the weight's gradient, as 0 times infinity is no number.
    """
    z_loss = float(z_loss)
    _check("linear_cross_entropy", x, weight, reduction)
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"targets must be {tuple(x.shape[:-1])}, got {tuple(targets.shape)}")
    _index64("targets", targets)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"ignore_index must fit 64 bits, got {ignore_index}")
    if not 0.0 <= z_loss < math.inf:
        raise ValueError(f"z_loss must be finite and not negative, got {z_loss}")
    return _loss(x, weight, targets, None, _Loss(reduction, z_loss=z_loss, ignore_index=int(ignore_index)))


def linear_distillation(x: torch.Tensor, weight: torch.Tensor, teacher_indices: torch.Tensor, teacher_logits: torch.Tensor, *,
                        temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """``temperature^2 sum_k p_k (log p_k - log q[i_k])`` for each token: q = softmax(x @ weight / temperature) over the
    vocabulary, p = softmax(teacher_logits / temperature) over the teacher's entries of the token, i their classes.

    Args:
        x, weight: as ``linear_cross_entropy``'s.
        teacher_indices: [..., K] int32 or int64, 1 <= K <= 1024, the classes of the teacher's entries in any order;
            negative ones are empty places.  A class that is there twice is two entries of the sum; one of V or more
            makes its token's loss and gradient NaN.
        teacher_logits: [..., K] float32 or bfloat16; p is their softmax over the token's entries (those of -inf left
            out; one of +inf or NaN makes the token's loss and gradient NaN).  The teacher gets no gradient.
        temperature: of both distributions.
        reduction: "mean" over the tokens that have an entry (0 if none has), "sum", or "none".

    Returns:
        The loss, float32: a scalar, or [...] for "none".  Differentiable (once) in x and weight.
    """
    temperature = float(temperature)
    _check("linear_distillation", x, weight, reduction)
    shape = teacher_indices.shape
    if len(shape) != x.dim() or shape[:-1] != x.shape[:-1] or teacher_logits.shape != shape:
        raise ValueError(f"teacher_indices and teacher_logits must be {(*x.shape[:-1], 'K')}, got {tuple(shape)} and "
                         f"{tuple(teacher_logits.shape)}")
    if not 1 <= shape[-1] <= MAX_ENTRIES:
        raise ValueError(f"a token has 1 to {MAX_ENTRIES} entries, got {shape[-1]}")
    _index64("teacher_indices", teacher_indices)
    if teacher_logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"teacher_logits must be float32 or bfloat16, got {teacher_logits.dtype}")
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError(f"temperature must be between 1e-3 and 1e3, got {temperature}")
    return _loss(x, weight, teacher_indices, teacher_logits.detach(), _Loss(reduction, temperature=temperature))
