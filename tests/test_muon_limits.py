"""How far "half" results may be off, whatever the groups of steps: 1.5 times what the oracle's roundings leave.

The inputs are float32 and so are the results, so nothing but the operator's own roundings is seen.  The limits are
numbers, not figures of the present schedule: a grouping that loses accuracy does not raise them.  Left out of the
oracle, the diagonals that are kept apart or what X loses in f16 pass them where a case names it, which shows that the
GPU tests would see their loss.  Products are in 64 bits in the oracle; float32 sums add 2e-6 at full rank to 1e-4 at rank 1,
a hundredth of the limits.
"""
from __future__ import annotations

import pytest
import torch
from test_muon_groups import gradient, rows

from mintext_amd.kernels.muon import COEFFICIENTS
from oracle import muon_oracle as O

# (op, M, N, rank): limit, and what has to pass it when it is left out
LIMITS = {
    ("newton_schulz", 64, 200, 8): (8e-3, ("remainder",)),
    ("newton_schulz", 128, 512, 1): (1.25e-2, ("diagonal", "remainder")),
    ("newton_schulz", 128, 512, 2): (6.8e-3, ("diagonal", "remainder")),
    ("newton_schulz", 100, 256, 32): (4.3e-3, ("remainder",)),
    ("newton_schulz", 200, 300, 32): (2.2e-3, ("remainder",)),
    ("newton_schulz", 256, 1024, 8): (2.8e-3, ("remainder",)),
    ("newton_schulz", 333, 1001, 600): (1.02e-3, ("remainder",)),
    ("newton_schulz", 704, 504, 100): (1.5e-3, ("remainder",)),
    ("newton_schulz", 300, 264, 32): (2.1e-3, ("remainder",)),
    ("muon_update", 128, 512, 2): (6.8e-3, ("diagonal", "remainder")),
    ("muon_update", 256, 1024, 2): (1e-2, ("diagonal", "remainder")),
    ("muon_update", 333, 1001, 8): (4.8e-3, ("diagonal", "remainder")),
    ("muon_update", 704, 504, 32): (3.9e-3, ("diagonal", "remainder")),
    ("muon_update", 200, 300, 100): (5.4e-3, ("remainder",)),
}


def off(got, want):
    return float((got - want).norm() / want.norm())


def group_of(op, M, N):
    if min(M, N) <= 128:
        return 3
    return 1 if op == "newton_schulz" or max(M, N) <= 1.25 * min(M, N) else 3


@pytest.mark.parametrize("case", LIMITS, ids=lambda c: "-".join(map(str, c)))
def test_the_oracle_keeps_them_and_a_loss_does_not(case):
    op, M, N, rank = case
    limit, needed = LIMITS[case]
    x = gradient(M, N, rank)
    want = O.newton_schulz(x, [COEFFICIENTS] * 5)
    schedule = rows(5, COEFFICIENTS, group_of(op, M, N))
    assert limit / 1.7 <= off(O.chain(x, schedule, 1), want) <= limit / 1.4
    for what in needed:
        assert off(O.chain(x, schedule, 1, lose=(what,)), want) > 1.1 * limit, what


def orthogonalised(op, x):
    from mintext_amd.kernels import muon_update, newton_schulz

    if op == "newton_schulz":
        return newton_schulz(x, precision="half")
    # a step from zeros that keeps nothing but the orthogonalised gradient
    return muon_update(torch.zeros_like(x), x, torch.zeros_like(x), lr=1.0, beta=0.0, scale=-1.0, precision="half")


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [1, 40])  # tiles of 64 x 64, and larger ones where there are many matrices
@pytest.mark.parametrize("case", LIMITS, ids=lambda c: "-".join(map(str, c)))
def test_the_operator_keeps_them(dev, case, copies):
    op, M, N, rank = case
    x = gradient(M, N, rank)
    want = O.newton_schulz(x, [COEFFICIENTS] * 5)
    got = orthogonalised(op, x.to(dev).expand(copies, M, N).contiguous()).double().cpu()
    assert torch.equal(got, got[:1].expand_as(got))
    assert off(got[0], want) <= LIMITS[case][0]


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(152, 472, 941), (1216, 384, 3143), (168, 1584, 335), (256, 1024, 100), (300, 700, 32)])
def test_bfloat16_results_are_little_more_than_rounded(dev, size):
    """The rounding of a bfloat16 result and 1.5 times the oracle's error with single steps, which are independent; in
    groups of two the second alone was as large as the first."""
    from mintext_amd.kernels import newton_schulz

    x = gradient(*size).bfloat16()
    want = O.newton_schulz(x, [COEFFICIENTS] * 5)
    own = off(O.chain(x, rows(5, COEFFICIENTS, 1), 1), want)
    rounding = off(want.bfloat16().double(), want)
    assert off(newton_schulz(x.to(dev)).double().cpu(), want) <= ((1.5 * own) ** 2 + rounding ** 2) ** 0.5
