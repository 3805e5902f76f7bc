"""What the gradients of the head's losses hold beside their results, over the admitted sizes (host only)."""
from __future__ import annotations

import pytest

from mintext_amd import _lib as L

MOST = 65535 * 64  # tokens, and columns


def up(n, m):
    return (n + m - 1) // m * m


@pytest.mark.parametrize("T, D, V", [(1, 64, 1000), (64, 4096, 131072), (65, 2048, 50257), (4096, 1001, 32000), (65536, 4096, 262144),
                                     (65537, 2049, 151936), (800000, 64, 32000), (1670000, 40, 50257), (MOST, 8, 1000),
                                     (MOST, 72, 131072), (MOST, 33, 4099), (300, 65, MOST)])
@pytest.mark.parametrize("order", [L.MTX_HEAD_DV, L.MTX_HEAD_VD])
@pytest.mark.parametrize("dtype", [L.MTX_BF16, L.MTX_F32])
def test_workspace_of_the_gradients(dtype, order, T, D, V):
    """1 GiB of the logits' gradient, or 320 columns of it where that is more; up to 64 tokens in bfloat16 two planes of it; x and a
    piece's gradient of the weight in float32, 16 times at most; bfloat16 copies of x and of 256 MiB, or 256 classes, of the weight."""
    size, few = (4, False) if dtype == L.MTX_F32 else (2, T <= 64)
    planes = 2 if few else 1
    dz = max(1 << 30, 320 * planes * T * size)
    sums = 16 * planes * T * up(D, 8) * 4
    piece = min(up(V, 256), max(256, dz // (planes * T * size)))
    sums += 16 * up(D, 8) * piece * 4
    copies = 0 if size == 4 else planes * T * up(D, 64) * 2 + max(256 << 20, 256 * up(D, 64) * 2)
    held = L.lib().mtx_head_loss_workspace_size(dtype, T, D, V, order, 1)
    assert 0 < held <= dz + sums + copies + 4096
    # of many tokens no sums are kept apart: dx in float32 once
    if T >= 800000:
        assert held <= dz + T * up(D, 8) * 4 + copies + 16 * up(D, 8) * 768 * 4 + 4096
