"""What the package offers at its root (host only)."""
from __future__ import annotations

import mintext_amd
from mintext_amd import kernels


def test_operators_of_the_kernels_package_are_at_the_root():
    """All but swiglu, the plain activation, and two helpers."""
    helpers = {"swiglu", "_sort_with_vjp", "update_expert_bias"}
    for name in set(kernels.__all__) - helpers:
        assert name in mintext_amd.__all__, name
        assert getattr(mintext_amd, name) is getattr(kernels, name)


def test_exported_names_exist():
    for module in (mintext_amd, kernels):
        assert len(set(module.__all__)) == len(module.__all__)
        for name in module.__all__:
            assert hasattr(module, name), name
