"""Where groups of steps end, and what the roundings between products leave of the result (host only: the oracle)."""
from __future__ import annotations

import pytest
import torch

from mintext_amd.kernels.muon import COEFFICIENTS, _schedule
from oracle import muon_oracle as O

# Triples that lift small singular values faster than the default ones.
STEEP = ((8.2872, -23.5959, 17.3004), (4.1071, -2.9478, 0.5448), (3.9487, -2.9089, 0.5518), (3.3184, -2.4885, 0.5100),
         (2.3007, -1.6689, 0.4188))


def rows(steps, coefficients, group):
    s = list(_schedule(steps, coefficients, group))
    return [tuple(s[9 * i:9 * i + 9]) for i in range(steps)]


def sizes(schedule):
    out, n = [], 0
    for row in schedule:
        n += 1
        if row[8]:
            out.append(n)
            n = 0
    return out


def gradient(M, N, rank):
    g = torch.Generator().manual_seed(7 * M + N + rank)
    x = torch.randn(M, rank, generator=g) * torch.exp(torch.randn(1, rank, generator=g))
    return x @ torch.randn(rank, N, generator=g)


@pytest.mark.parametrize("coefficients", [COEFFICIENTS, (1.5, -0.5, 0.0), (3.0, -3.2, 1.2), (1.0, 0.0, 0.0)])
@pytest.mark.parametrize("group", [1, 2, 3])
def test_gentle_coefficients_fill_the_groups(group, coefficients):
    for steps in range(1, 12):
        most = -(-steps // group)
        assert sizes(rows(steps, coefficients, group)) == [steps // most + (g < steps % most) for g in range(most)]


@pytest.mark.parametrize("group", [1, 2, 3])
def test_steep_coefficients_end_groups_early(group):
    schedule = rows(5, STEEP, group)
    growth, first = 1.0, True
    for row in schedule:
        growth = row[0] if first else growth * row[0]  # what small singular values grow by since the Gram product
        assert first or growth <= 1.01 * COEFFICIENTS[0] ** group
        assert not first or row[6] == row[4]           # P is Q at a group's first step
        first = bool(row[8])
    assert first and sum(sizes(schedule)) == 5


@pytest.mark.parametrize("precision", [1, 2])
@pytest.mark.parametrize("size", [(256, 1024, 8), (256, 1024, 100), (300, 264, 600), (128, 512, 8)])
def test_steep_coefficients_are_no_worse_in_groups(size, precision):
    """A group's error comes with the square of its growth; where that is held to what the default triples reach, groups
    cost no more than with those, which is up to four times the single steps' error (256 x 1024, rank 100, in threes)."""
    x = gradient(*size)
    want = O.newton_schulz(x, STEEP)
    off = lambda group: float((O.chain(x, rows(5, STEEP, group), precision) - want).norm() / want.norm())
    assert max(off(2), off(3)) <= 4 * off(1)


def test_the_oracle_without_roundings_is_the_definition():
    x = gradient(48, 80, 60)
    want = O.newton_schulz(x, [COEFFICIENTS] * 5)
    off = (O.chain(x, rows(5, COEFFICIENTS, 3), 2) - want).norm() / want.norm()
    assert 0 < off < 1e-5
