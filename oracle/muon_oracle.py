"""CPU oracle of the orthogonalised updates: the quintic in 64 bits, and the chain of products with the roundings of
what is stored on the way.

``newton_schulz`` is the definition: X = x / (|x|_F + eps), then X <- a X + (b A + c A^2) X with A = X X^T on the smaller
side (the products of the reference's optimiser, mintext/optim/optimizer.py:92-168).

``chain`` computes the same in groups of steps, each one Gram product, symmetric S x S products and one product with X, and
rounds every matrix as it is held between products: in one f16 plane (``planes`` 1) or in two, the diagonals of Q and P and
what X loses in f16 apart.  Products are in 64 bits: what float32 sums add is a hundredth of one plane's roundings.
``lose`` leaves out what is kept apart, which says how much of the error it takes away: "diagonal" (what f16 loses of the diagonals of Q and P), "remainder" (what it loses of X).
"""
from __future__ import annotations

import math

import torch

SMALL = 128  # matrices of up to that many rows or columns have two planes within a group in any case


def newton_schulz(x, triples, eps=1e-7):
    x = x.double()
    x = x / (x.square().sum().sqrt() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for a, b, c in triples:
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


def _f16(t):
    r = t.to(torch.float16).double()
    assert torch.isfinite(r).all(), "a matrix left f16's range"
    return r


class _Held:
    """A matrix as it is held: ``m``, in true units, and beside it in ``rest`` what f16 loses of its diagonal."""

    def __init__(self, t, scale, planes, apart=False, lose=()):
        self.m = _f16(t * scale)
        if planes == 2:
            self.m = self.m + _f16(t * scale - self.m)
        self.rest, self.diagonal = torch.zeros(len(t), dtype=t.dtype), self.m.diagonal() / scale
        if apart and "diagonal" not in lose:
            self.rest = _f16(t.diagonal() * scale - self.m.diagonal()) / scale
            self.diagonal = t.diagonal().float().double()
        self.m = self.m / scale

    def times(self, other):
        """What the diagonals lost times each other is left out."""
        return self.m @ other.m + self.rest[:, None] * other.m + self.m * other.rest[None]


def chain(x, schedule, planes, eps=1e-7, lose=()):
    """``x`` [M, N], float32 or bfloat16; ``schedule``: rows (a, b, c, scales of A, Q, T, P and X, whether the group ends)."""
    tall = x.shape[0] > x.shape[1]
    x = (x.t() if tall else x).double().contiguous()
    eye = torch.eye(len(x), dtype=x.dtype)
    inner = 2 if len(x) <= SMALL else planes

    def hold_x(x, scale, first):
        """X as the products see it, and what that lacks: 8-bit floats, or (in two planes only of the first X) f16."""
        hi = _f16(x * scale)
        if planes == 2:
            hi = hi + _f16(x * scale - hi)
        lack = x * scale - hi
        lack = lack.to(torch.float8_e5m2).double() if planes == 1 else _f16(lack) if first else torch.zeros_like(lack)
        return hi / scale, torch.zeros_like(lack) if "remainder" in lose else lack / scale

    norm = float(x.square().sum().sqrt()) + eps
    x, lack = hold_x(x / norm, norm * 2.0 ** (13 - math.floor(math.log2(norm))), True)
    A = None
    for i, (a, b, c, sa, sq, st, sp, sx, ends) in enumerate(schedule):
        if A is None:
            A, P = _Held(x @ x.t(), sa, inner), None
        Q = _Held(a * eye + b * A.m + c * (A.m @ A.m), sq, planes if P is None and ends else inner, True, lose)
        if P is not None:
            P = _Held(Q.times(P), sp, planes if ends else inner, True, lose)
        else:
            P = Q
        if ends:
            y = P.m @ x + P.rest[:, None] * x + P.diagonal[:, None] * lack
            x, lack = hold_x(y, sx, False) if i + 1 < len(schedule) else (y, None)
            A = None
        else:
            A = _Held(Q.times(_Held(Q.times(A), st, inner)), schedule[i + 1][3], inner)
    return x.t() if tall else x
