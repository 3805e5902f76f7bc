"""Coefficients and numbers of steps other than the default ones where products run launch by launch (above 128 rows).

Two bounds.  The oracle computes the same products with the roundings of what is stored, by the same schedule; the
operator may be 1.5 times as far from the definition in 64 bits ("half").  In "full" float32 sums count for more than
what is stored, so there each product of n terms is disturbed by random signs times (4 + sqrt n) 2^-24 of its terms'
sizes, as in the tests of the default coefficients, and the changes of the result are added up.
"""
from __future__ import annotations

import pytest
import torch
from test_gpu_muon import held
from test_muon_groups import STEEP, gradient
from test_muon_limits import off

from mintext_amd.kernels.muon import COEFFICIENTS, _schedule
from oracle import muon_oracle as O

pytestmark = pytest.mark.gpu

CUBIC = (1.5, -0.5, 0.0)         # no product squares A
FAINT = (1.0, -1e-3, 1e-6)       # the product that does cannot carry b A in f16
EVEN = (1.25, 0.0, -0.25)        # nothing to carry
MIXED = ((1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.0, -1e-3, 1e-6), (1.5, -0.5, 0.0), (3.4445, -4.7750, 2.0315),
         (1.25, 0.0, -0.25), (1.9, -1.2, 0.3))
SIZES = [(200, 300, 400), (333, 150, 100)]  # rows off a multiple of 32, wide and tall, long enough for groups


def triples(coefficients, steps):
    return list(coefficients[:steps]) if isinstance(coefficients[0], tuple) else [coefficients] * steps


def oracle_error(x, want, coefficients, steps, group):
    s = list(_schedule(steps, coefficients, group))
    return off(O.chain(x, [tuple(s[9 * i:9 * i + 9]) for i in range(steps)], 1), want)


@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("copies", [1, 64])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7])
@pytest.mark.parametrize("coefficients", [CUBIC, FAINT, EVEN, MIXED, COEFFICIENTS],
                         ids=["cubic", "faint", "even", "mixed", "default"])
def test_newton_schulz(dev, coefficients, steps, size, copies, precision):
    from mintext_amd.kernels import newton_schulz

    c = coefficients[:steps] if isinstance(coefficients[0], tuple) else coefficients
    x = gradient(*size)
    got = newton_schulz(x.to(dev).expand(copies, *x.shape).contiguous(), steps, coefficients=c, precision=precision)
    assert torch.equal(got, got[:1].expand_as(got))
    if precision == "full":
        held(got[:1], x[None].to(dev), True, 2.0 ** -24, steps=steps, coef=c)
    else:
        want = O.newton_schulz(x, triples(c, steps))
        assert off(got[0].double().cpu(), want) <= 1.5 * oracle_error(x, want, c, steps, 1) + 2.0 ** -24


@pytest.mark.parametrize("steps", [2, 3, 4, 5, 7])
@pytest.mark.parametrize("coefficients", [CUBIC, FAINT, EVEN, MIXED, STEEP], ids=["cubic", "faint", "even", "mixed", "steep"])
@pytest.mark.parametrize("size", [*SIZES, (256, 1024, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_muon_update(dev, coefficients, size, dtype, steps):
    """Groups of up to three."""
    from mintext_amd.kernels import muon_update

    steps = min(steps, 5) if coefficients is STEEP else steps
    c = coefficients[:steps] if isinstance(coefficients[0], tuple) else coefficients
    x = gradient(*size)
    g = torch.Generator().manual_seed(3)
    p = (torch.randn(x.shape, generator=g) * 0.02).to(dtype)
    got = p.to(dev)
    muon_update(got, x.to(dev), torch.zeros(x.shape, device=dev), lr=0.5, beta=0.0, scale=1.0, steps=steps, coefficients=c,
                precision="half")
    o = O.newton_schulz(x, triples(c, steps))
    want = p.double() - 0.5 * o
    rounding = (torch.finfo(dtype).eps / 2 + 2.0 ** -22) * want.norm()  # of the weights, at most half a step each
    assert (got.double().cpu() - want).norm() <= 0.5 * 1.5 * oracle_error(x, o, c, steps, 3) * o.norm() + rounding
    if coefficients is STEEP and steps == 5 and size == (256, 1024, 8):
        # in groups as long as the default ones the error was 8 % of the orthogonalised gradient; the weights' rounding,
        # 2^-8 |w| = 0.04 at most in bfloat16, is more than 1 % of it (0.014) and less than 8 % (0.11)
        assert (got.double().cpu() - want).norm() <= 0.5 * 0.01 * o.norm() + rounding
