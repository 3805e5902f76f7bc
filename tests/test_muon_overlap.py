"""Operands of ``muon_update`` that share memory are refused, those that lie between each other are not (host only)."""
from __future__ import annotations

import random

import pytest
import torch

from mintext_amd.kernels import muon_update
from mintext_amd.kernels.muon import _overlap, _writable


def stack(flat, start, E, M, N, batch, row):
    return flat.as_strided((E, M, N), (batch, row, 1), start)


def bytes_of(t):
    E, M, N = t.shape
    size, start = t.element_size(), t.data_ptr()
    return {start + (e * t.stride(0) + m * t.stride(1) + n) * size + k
            for e in range(E) for m in range(M) for n in range(N) for k in range(size)}


@pytest.mark.parametrize("seed", range(8))
def test_against_the_bytes_themselves(seed):
    rng = random.Random(seed)
    flat = torch.zeros(4096)
    seen = [0, 0]
    while min(seen) < 60:
        E, M, N = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 5)
        row = rng.randint(N, 2 * N + 2)
        batch = rng.randint((M - 1) * row + N, (M - 1) * row + 3 * N)
        if rng.random() < 0.3:  # matrices between each other's rows
            batch = rng.randint(N, 2 * N)
            row = (E - 1) * batch + N + rng.randint(0, N)
        both = [flat, flat.view(torch.bfloat16) if rng.random() < 0.3 else flat]
        rng.shuffle(both)
        scale = [f.element_size() // min(g.element_size() for g in both) for f in both]
        if any(s != 1 for s in scale):  # the same bytes from row to row
            row, batch = 2 * row, 2 * batch
        a, b = (stack(f, rng.randint(0, 60 // s), E, M, N, batch // s, row // s) for f, s in zip(both, scale))
        _writable(a, "a"), _writable(b, "b")
        want = bool(bytes_of(a) & bytes_of(b))
        assert _overlap(a, b) == _overlap(b, a) == want, (a.shape, a.stride(), b.stride(), a.data_ptr() - b.data_ptr())
        seen[want] += 1


@pytest.mark.parametrize("seed", range(4))
def test_other_strides_are_never_let_through(seed):
    rng = random.Random(seed)
    flat = torch.zeros(4096)
    shared = 0
    while shared < 60:
        E, M, N = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 5)
        made = []
        for k in range(2):
            row = rng.randint(N, 2 * N + 2)
            least = 0 if k else (M - 1) * row + N  # the second may be a gradient of any strides
            made.append(stack(flat, rng.randint(0, 40), E, M, N, rng.randint(least, (M - 1) * row + 3 * N), row))
        if bytes_of(made[0]) & bytes_of(made[1]):
            assert _overlap(*made)
            shared += 1


def test_shifted_operands_are_refused():
    flat = torch.zeros(3 * 4 * 8 + 8)
    a, b, c = flat[:96].view(3, 4, 8), flat[8:].view(3, 4, 8), torch.zeros(3, 4, 8)
    for operands in ((a, b, c), (b, a, c), (a, c, b), (b, c, a), (c, a, b), (c, b, a)):
        with pytest.raises(ValueError, match="share memory"):
            muon_update(*operands, lr=0.1)
    fused = torch.zeros(3, 4, 24)
    for columns in (slice(7, 15), slice(1, 9)):
        with pytest.raises(ValueError, match="share memory"):
            muon_update(fused[..., :8], fused[..., columns], c, lr=0.1)


def test_neighbours_are_accepted():
    """Up to the device."""
    fused = torch.zeros(3, 4, 24)
    flat = torch.zeros(3 * 96)
    for operands in ((fused[..., :8], fused[..., 8:16], fused[..., 16:]), flat.view(3, 3, 4, 8).unbind(),
                     (torch.zeros(3, 4, 8), torch.zeros(1, 4, 8).expand(3, 4, 8), torch.zeros(3, 4, 8)),
                     fused.view(3, 4, 3, 8).unbind(2)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            muon_update(*operands, lr=0.1)
