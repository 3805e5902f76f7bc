"""Orthogonalised updates of (stacked) weight matrices: Newton-Schulz products and the Muon step.

The optimiser side of ``tgmm``'s weight gradients (the reference's optimiser runs Muon with dimension numbers for the
experts' stacks, mintext/optim/optimizer.py:92-168): every matrix of a stack [..., M, N] is orthogonalised by itself,
all of them in the same launches.

``newton_schulz`` maps the singular values of ``x / (|x|_F + eps)`` by ``steps`` odd quintics a s + b s^3 + c s^5, which
brings them near 1 and keeps the singular vectors.  ``muon_update`` does an optimiser step in place:

    m <- beta m + (1 - beta) g;   u = (1 - beta) g + beta m (Nesterov) or m
    w <- (1 - lr weight_decay) w - lr factor newton_schulz(u)

Precision.  "half" and "full" run on the 16-bit matrix cores with float32 sums: "half" holds the matrices between products
in f16 (11 bits, under power-of-two scales that their bounded singular values allow), "full" in two f16 planes (22 bits,
three times the products).  "double" is float64 throughout, on the float64 matrix cores.  Rounding errors in directions
in which x is nearly singular grow as those do, by |a| a step, so that what a result is off by depends on x's rank.  Five
steps with the default coefficients are off, before the result is rounded to its type, by (2-norm)

    "half"    0.04 to 0.17 % for bfloat16 in newton_schulz; 0.04 to 0.5 % in muon_update, which takes steps in groups,
              and for float32 x; up to 1.4 % in those for ranks of 4 and less
    "full"    2e-6 at full rank to 4e-5 at rank 8, up to 1.3e-4 below: what products in float32 throughout come to
    "double"  1e-11

More or steeper steps end further off.  ``newton_schulz`` takes "double" for float32 and "half" for bfloat16, whose own
rounding is as coarse; ``muon_update``, where the result is a small change of the weights, "full" for float32 weights and
"half" for bfloat16.  The Frobenius norm is summed in float64 and momentum is float32.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .. import _lib as L

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
# Steps between two Gram products, at most, by planes: fewer products with more, smaller errors with fewer (128 x 768 x 2048 in
# bfloat16, five steps: 4.07 ms by themselves, 3.46 in twos, 3.30 in threes).  A result in "half" takes single steps, which
# leave it little more than its rounding to bfloat16 off, 1.75e-3 for 1.66e-3 (twos 2.0 to 2.7e-3); in "full" float32 sums
# count for more than the groups, and a small change of weights stands threes.  Matrices of _SMALL or less on a side take
# threes in any case: their products in between are held in 22 bits (64 x 128 x 1408 in "full" 212 us, 265 in twos).  Those
# near square gain nothing from groups, whose symmetric products cost what the others save: one of 2048 x 2048 takes
# 366 us in single steps, 405 in twos, 419 in threes; 8 of 1024 x 1280 445, 446, 440; 128 of 768 x 1152 3.02 ms, 2.85, 2.71.
_GROUP_RESULT, _GROUP_STEP, _SMALL, _SQUARE = {1: 1, 2: 2}, {1: 3, 2: 3}, 128, 1.25
# What a Gram product's rounding becomes grows with the square of the group's product of polynomials, so a group ends early
# where that product would pass what as many steps with the coefficients above reach: steeper ones (8.3, 4.1, 3.9, ..)
# in threes end 8 % off at rank 8 of 256 x 1024 in "half", 0.4 % this way, as by themselves (simulated roundings).
_GROWTH = 3.45
_PLANES = {"half": 1, "full": 2, "double": L.MTX_NS_F64}


@functools.lru_cache(maxsize=64)
def _schedule(steps: int, coefficients: tuple, group: int):
    """The 9 floats a step of ``mtx_newton_schulz``: coefficients, scales, and where a group of steps ends.

    The singular values start in [0, 1] (the Frobenius norm bounds them), so those of every matrix on the way have a
    bound; an entry is at most its matrix's largest singular value.  Each scale is the largest power of two that
    keeps 1.25 times the bound inside f16.
    """
    triples = [coefficients] * steps if not isinstance(coefficients[0], tuple) else list(coefficients)
    groups = -(-steps // group)
    sizes = [steps // groups + (g < steps % groups) for g in range(groups)]
    last = [sum(sizes[:g + 1]) - 1 for g in range(groups)]

    def scale(bound):
        if not bound < 2.0 ** 12:
            raise ValueError("these coefficients let singular values in [0, 1] grow out of range")
        return 2.0 ** min(20, math.floor(math.log2(60000 / (1.25 * max(bound, 2.0 ** -8)))))

    top, flat, first = 1.0, [], True
    for i, (a, b, c) in enumerate(triples):
        quintic = lambda s: [a + b * t * t + c * t ** 4 for t in s]
        if not first:
            q = quintic(s)
            p = [u * v for u, v in zip(p, q)]
            if max(abs(v) for v in p) > _GROWTH ** group:
                flat[-1], first = 1.0, True
        if first:
            s = [top * k / 2048 for k in range(2049)]
            q = p = quintic(s)
        bound_t = max(abs(v) * t * t for v, t in zip(q, s))
        sq = scale(max(abs(v) for v in q))
        sa = scale(max(t * t for t in s))
        if 0 < abs(b) < 100 * abs(c):  # the product that squares A carries b as (b / c) sa, in f16 as well
            sa = min(sa, 2.0 ** math.floor(math.log2(60000 * abs(c / b))))
        flat += [a, b, c, sa, sq, scale(bound_t),
                 sq if first else scale(max(abs(v) for v in p)), 0.0, float(i in last)]
        s = [abs(v) * t for v, t in zip(q, s)]
        top = max(s)
        flat[-2] = scale(top)
        first = i in last
    return (ctypes.c_float * len(flat))(*flat)


@functools.lru_cache(maxsize=64)
def _schedule64(steps: int, coefficients: tuple):
    """The same for float64, whose range needs no scales: in their place what float32 loses of the coefficients."""
    _schedule(steps, coefficients, 1)  # refuses coefficients that diverge
    triples = [coefficients] * steps if not isinstance(coefficients[0], tuple) else coefficients
    single = lambda v: ctypes.c_float(v).value
    flat = [v for c in triples for v in (*map(single, c), *(v - single(v) for v in c), 0.0, 0.0, 0.0)]
    return (ctypes.c_float * len(flat))(*flat)


def _arguments(steps, coefficients, eps, precision, t, groups, single):
    """(schedule, planes); ``groups``: the longest, by planes; ``single``: the precision of what is float32."""
    if not isinstance(steps, int) or not 1 <= steps <= 64:
        raise ValueError(f"steps must be an int from 1 to 64, got {steps!r}")
    if not eps > 0:
        raise ValueError(f"eps must be positive, got {eps!r}")
    if precision not in (None, *_PLANES):
        raise ValueError(f'precision must be "half", "full", "double" or None, got {precision!r}')
    try:
        if isinstance(coefficients[0], (tuple, list)):
            c = tuple(tuple(float(v) for v in t) for t in coefficients)
            good = len(c) == steps and all(len(t) == 3 for t in c)
        else:
            c = tuple(float(v) for v in coefficients)
            good = len(c) == 3
    except (TypeError, IndexError):
        good = False
    if not good or not all(math.isfinite(v) for t in c for v in (t if isinstance(t, tuple) else (t,))):
        raise ValueError("coefficients must be three finite numbers, or three for each step")
    planes = _PLANES[precision or (single if t.dtype == torch.float32 else "half")]
    if planes == L.MTX_NS_F64:
        return _schedule64(steps, c), planes
    group = groups[planes]
    if min(t.shape[-2:]) <= _SMALL:
        group = 3
    elif max(t.shape[-2:]) <= _SQUARE * min(t.shape[-2:]):
        group = 1
    return _schedule(steps, c, group), planes


def _check_stack(t: torch.Tensor, name: str):
    if t.dim() < 2:
        raise ValueError(f"{name} must be a matrix or a stack of them, got {tuple(t.shape)}")
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")


def _readable(t: torch.Tensor) -> torch.Tensor:
    """As [E, M, N] with rows of consecutive elements, copied where it has to be."""
    M, N = t.shape[-2:]
    t = t.reshape(math.prod(t.shape[:-2]), M, N)
    if t.numel() == 0 or (t.stride(2) == 1 or N == 1) and (t.stride(1) >= N or M == 1):
        return t
    return t.contiguous()


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """(batch, row) of a [E, M, N] stack; what a size of 1 never uses is set to what dense storage has."""
    E, M, N = t.shape
    row = t.stride(1) if M > 1 else N
    return (t.stride(0) if E > 1 else M * row), row


def _writable(t: torch.Tensor, name: str) -> torch.Tensor:
    """As [E, M, N] without a copy, its elements apart from each other."""
    M, N = t.shape[-2:]
    E = math.prod(t.shape[:-2])
    if t.numel() == 0:
        return t.reshape(E, M, N)
    try:
        v = t.detach().view(E, M, N)
    except RuntimeError:
        raise ValueError(f"{name} is updated in place: its leading dimensions must be mergeable into one") from None
    batch, row = _strides(v)
    apart = batch >= (M - 1) * row + N or row >= (E - 1) * batch + N and batch >= N
    if (v.stride(2) != 1 and N > 1) or row < N or (E > 1 and not apart):
        raise ValueError(f"{name} is updated in place: it needs rows of consecutive elements that do not overlap")
    return v


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses from the first byte of a [E, M, N] stack to behind its last."""
    E, M, N = t.shape
    batch, row = _strides(t)
    start = t.data_ptr()
    return start, start + ((E - 1) * batch + (M - 1) * row + N) * t.element_size() if t.numel() else start


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [E, M, N] stacks, of which one is as ``_writable`` returns it, share memory.  Stacks that lie between
    each other's rows with the same strides (halves of a fused buffer) do not; with others they count as sharing it."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0 or a0 == a1 or b0 == b1:
        return False
    E, M, N = a.shape
    da, db = ([s * t.element_size() for s in _strides(t)] for t in (a, b))
    na, nb = N * a.element_size(), N * b.element_size()
    apart = b0 - a0
    steps = [(d, n) for d, e, n in zip(da, db, (E, M)) if n > 1]
    if any(d != e for d, e, n in zip(da, db, (E, M)) if n > 1):
        return True
    # Is there a whole combination of the strides that brings a row of b to a row of a?  The smaller stride's reach lies
    # within the larger one, so that each has two candidates.
    steps.sort(reverse=True)
    reach = max(na, nb)
    for d, n in reversed(steps):
        if reach > d:
            return True
        reach += (n - 1) * d
    rests = [apart]
    for d, n in steps:
        rests = [r - k * d for r in rests for k in (r // d, r // d + 1) if abs(k) < n]
    return any(-nb < r < na for r in rests)


def newton_schulz(x: torch.Tensor, steps: int = 5, *, coefficients=COEFFICIENTS, eps: float = 1e-7,
                  precision: str | None = None) -> torch.Tensor:
    """Orthogonalise each matrix of ``x`` [..., M, N] by ``steps`` Newton-Schulz products.

    X <- x / (|x|_F + eps), then ``steps`` times X <- a X + (b A + c A^2) X with A = X X^T.  A matrix of zeros stays
    zeros; one that holds a NaN or an infinity becomes NaN, without touching the others.

    Args:
        x: float32 or bfloat16, any strides (rows that are not consecutive elements are copied first).
        coefficients: (a, b, c), or such a triple for each step.
        precision: "half", "full", "double" or None, by x's dtype (see the module).

    Returns:
        a dense tensor of x's shape and dtype.  Not differentiable: an x that requires a gradient or has a
        forward-mode tangent is refused, and so is a jit trace.
    """
    L.refuse_watched("newton_schulz", x)
    _check_stack(x, "x")
    sched, planes = _arguments(steps, coefficients, eps, precision, x, _GROUP_RESULT, "double")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("newton_schulz is not differentiable: pass x.detach()")
    dev = L.require_device(x)
    v = _readable(x)
    E, M, N = v.shape
    out = torch.empty((E, M, N), dtype=x.dtype, device=dev)
    ws = L.workspace(L.query("mtx_newton_schulz_workspace_size", E, M, N, planes), dev)
    with L.on_device(dev):
        L.call("mtx_newton_schulz", L.ptr(v), L.dtype_code(x.dtype), E, M, N, *_strides(v), sched, steps, eps, planes,
               L.ptr(out), M * N, N, L.ptr(ws), ws.numel(), L.stream(dev))
    return out.view(x.shape)


def muon_update(param: torch.Tensor, grad: torch.Tensor, momentum: torch.Tensor, *, lr, beta: float = 0.95,
                nesterov: bool = True, weight_decay: float = 0.0, scale: str | float = "spectral", steps: int = 5,
                coefficients=COEFFICIENTS, eps: float = 1e-7, precision: str | None = None) -> torch.Tensor:
    """One Muon step of a stack of weights, in place (formulas in the module's docstring).

    Args:
        param: [..., M, N] weights used as ``x @ param``, float32 or bfloat16; updated in place.  A view with rows of
            consecutive elements will do, e.g. the gate half ``gate_up[..., :I]`` of a fused stack.
        grad: its gradient, of the same shape, float32 or bfloat16.
        momentum: float32 of the same shape, updated in place (zeros before the first step).  The three must not share
            memory.
        lr: learning rate, a number or a float32 device tensor of one element (read when the step runs, so that a
            captured step follows it).
        scale: factor of the update: "spectral" sqrt(max(1, N / M)), "rms" 0.2 sqrt(max(M, N)), or a number.
        precision: as in ``newton_schulz``, by param's dtype.

    Returns:
        param.  A tensor with a forward-mode tangent is refused, and so is a jit trace.
    """
    L.refuse_watched("muon_update", param, grad, momentum, lr if isinstance(lr, torch.Tensor) else None)
    for t, name in ((param, "param"), (grad, "grad"), (momentum, "momentum")):
        _check_stack(t, name)
        if t.shape != param.shape:
            raise ValueError(f"{name} must have param's shape {tuple(param.shape)}, got {tuple(t.shape)}")
    if momentum.dtype != torch.float32:
        raise TypeError(f"momentum must be float32, got {momentum.dtype}")
    sched, planes = _arguments(steps, coefficients, eps, precision, param, _GROUP_STEP, "full")
    M, N = param.shape[-2:]
    if scale == "spectral":
        factor = math.sqrt(max(1.0, N / max(M, 1)))
    elif scale == "rms":
        factor = 0.2 * math.sqrt(max(M, N))
    elif isinstance(scale, (int, float)):
        factor = float(scale)
    else:
        raise ValueError(f'scale must be "spectral", "rms" or a number, got {scale!r}')
    lr_dev = None
    if isinstance(lr, torch.Tensor):
        if lr.dtype != torch.float32 or lr.numel() != 1:
            raise TypeError("lr must be a number or a float32 tensor of one element")
        lr, lr_dev = 0.0, lr
    p, m = _writable(param, "param"), _writable(momentum, "momentum")
    if param.numel() and len({param.data_ptr(), grad.data_ptr(), momentum.data_ptr()}) < 3:
        raise ValueError("param, grad and momentum must be three different tensors")
    g = _readable(grad.detach())
    spans = sorted(map(_span, (p, m, g)))
    if (spans[0][1] > spans[1][0] or spans[1][1] > spans[2][0]) and (_overlap(p, m) or _overlap(p, g) or _overlap(m, g)):
        raise ValueError("param, grad and momentum must not share memory")
    dev = L.require_device(param, grad, momentum, lr_dev)
    E = p.shape[0]
    ws = L.workspace(L.query("mtx_newton_schulz_workspace_size", E, M, N, planes), dev)
    with L.on_device(dev):
        L.call("mtx_muon_update", L.ptr(p), L.dtype_code(p.dtype), *_strides(p), L.ptr(g), L.dtype_code(g.dtype),
               *_strides(g), L.ptr(m), *_strides(m), E, M, N, beta, int(nesterov), lr, L.ptr(lr_dev), weight_decay, factor,
               sched, steps, eps, planes, L.ptr(ws), ws.numel(), L.stream(dev))
    torch.autograd.graph.increment_version([t for t in (param, momentum) if not t.is_inference()])
    return param
