"""MoE kernels: token routing and grouped matmul (mirror of mintext/kernels/__init__.py:3-6).

The reference exports route, unroute, grouped_matmul, grouped_matmul_vjp and tgmm; this
package adds route_topk (router top-k), grouped_matmul_swiglu (fused gate_up + SwiGLU),
swiglu, the blockwise-fp8 entry points in ``fp8``, linear (the dense product
with its epilogue), layer_norm and rms_norm, linear_cross_entropy and linear_distillation (losses of a
vocabulary-sized head without its logits in memory), and newton_schulz and muon_update (orthogonalised updates of expert weights).
"""
from .grouped_matmul import grouped_matmul, grouped_matmul_swiglu, grouped_matmul_vjp, swiglu, tgmm
from .head_loss import linear_cross_entropy, linear_distillation
from .linear import linear
from .moe_dispatch import _sort_with_vjp, route, unroute
from .muon import muon_update, newton_schulz
from .norm import layer_norm, rms_norm
from .router import route_topk, update_expert_bias

__all__ = ["route", "unroute", "grouped_matmul", "grouped_matmul_vjp", "tgmm", "route_topk",
           "grouped_matmul_swiglu", "swiglu", "linear", "layer_norm", "rms_norm", "linear_cross_entropy",
           "linear_distillation", "newton_schulz", "muon_update", "_sort_with_vjp", "update_expert_bias"]
