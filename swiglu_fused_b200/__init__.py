"""B200-native fused SwiGLU gate/up stage (sm_100a, tcgen05 + TMA).

Public surface = the reference's two operators::

    from swiglu_fused_b200 import matmul_silu_mul, matmul_fused_swiglu

The same functions are importable under the reference's own module paths,
``swiglu.matmul_silu_mul`` and ``swiglu.matmul_fused_swiglu``.  Beside them: the operators of a
mixture of SwiGLU experts (``experts``) and the differentiable forms (``autograd``, ``module``).
"""
from ._lib import TileConfig, SglError
from .autograd import fused_swiglu, fused_swiglu_experts
from .experts import (ExpertOrder, SavedExperts, SavedPreact, expert_combine, expert_combine_grad,
                      expert_dispatch, expert_order, experts_swiglu, experts_swiglu_backward,
                      experts_swiglu_save, experts_swiglu_workspace_bytes,
                      fused_swiglu_backward_saved,
                      grouped_fused_swiglu, grouped_fused_swiglu_save, grouped_grad_preact,
                      grouped_matmul, grouped_weight_grad, matmul_fused_swiglu_save_preact,
                      swiglu_grad_preact_saved)
from .module import PackedSwiGLUExperts, PackedSwiGLULinear
from .ops import (matmul_bf16, matmul_fused_swiglu, matmul_silu_mul, tune_matmul_fused_swiglu,
                  tune_matmul_silu_mul)

__all__ = [
    "matmul_silu_mul",
    "matmul_fused_swiglu",
    "matmul_bf16",
    "tune_matmul_silu_mul",
    "tune_matmul_fused_swiglu",
    "fused_swiglu",
    "fused_swiglu_experts",
    "expert_order",
    "expert_dispatch",
    "expert_combine",
    "expert_combine_grad",
    "grouped_fused_swiglu",
    "grouped_fused_swiglu_save",
    "grouped_matmul",
    "grouped_grad_preact",
    "grouped_weight_grad",
    "experts_swiglu",
    "experts_swiglu_workspace_bytes",
    "experts_swiglu_save",
    "experts_swiglu_backward",
    "matmul_fused_swiglu_save_preact",
    "swiglu_grad_preact_saved",
    "fused_swiglu_backward_saved",
    "ExpertOrder",
    "SavedPreact",
    "SavedExperts",
    "PackedSwiGLULinear",
    "PackedSwiGLUExperts",
    "TileConfig",
    "SglError",
]
