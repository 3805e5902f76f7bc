"""Few rows against weights of 128 MiB and more, which the kernel streams past the memory-side cache."""
from __future__ import annotations

import pytest
import torch
from conftest import launched
from test_gpu_linear import check

pytestmark = pytest.mark.gpu

K, N = 8200, 8264  # neither whole chunks of the reduction nor whole tiles of columns; 129 MiB of bf16


@pytest.mark.parametrize("rows", [1, 24, 61])
def test_streamed_weights(dev, rows):
    from mintext_amd.kernels import linear

    check(dev, rows, K, N, torch.bfloat16, "silu", True, True, False)
    check(dev, rows, K, N, torch.bfloat16, None, False, False, False, seed=1)
    x, w = torch.zeros(rows, K, device=dev).bfloat16(), torch.zeros(K, N, device=dev).bfloat16()
    blocks, waves = {1: (1, 8), 24: (2, 8), 61: (4, 4)}[rows]
    assert f"thin_kernel<{blocks}, {waves}, true>" in launched(lambda: linear(x, w))
