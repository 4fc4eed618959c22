"""``torch.autograd`` wiring of the stage for training.

Forward: the side-store kernel (h + factors in one launch).  Backward: the elementwise
kernel for ``grad_preact``, then ``grad_x = grad_preact @ W^T`` and
``grad_W = x^T @ grad_preact`` on the GEMM form of the same kernel, each reading its
transposed operand in place.  The reference keeps its autograd Functions in its Triton
module (``swiglu/triton/impls.py:2913-3369``) and runs the two GEMMs through cuBLAS
(``:100-124``).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .experts import (SavedExperts, SavedPreact, _checkpoint_bits, experts_swiglu_backward,
                      experts_swiglu_save, fused_swiglu_backward_saved,
                      matmul_fused_swiglu_save_preact)
from .ops import matmul_bf16, matmul_fused_swiglu_save_factors, swiglu_grad_preact


class FusedSwiGLUFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        h, factors = matmul_fused_swiglu_save_factors(x, w)
        ctx.save_for_backward(x, w, factors)
        return h

    @staticmethod
    def backward(ctx, grad_h: torch.Tensor):
        x, w, factors = ctx.saved_tensors
        # grad_preact overwrites the saved factors (no second [M, 2N] buffer).  The write goes
        # through a raw pointer, which autograd's version counter cannot see, so a second
        # backward over the same graph would silently multiply dy into factors that already
        # hold dy: refuse it instead.  (The reference writes grad_de to a new tensor and then
        # frees the saved ones, swiglu/triton/impls.py:3107-3116.)
        if getattr(ctx, "_factors_consumed", False):
            raise RuntimeError(
                "FusedSwiGLUFunction.backward ran twice over one forward: the saved factors "
                "were overwritten in place by the first backward (retain_graph=True is not "
                "supported; run the forward again)")
        ctx._factors_consumed = True
        grad_preact = swiglu_grad_preact(grad_h.contiguous(), factors, out=factors)  # in place
        grad_x = matmul_bf16(grad_preact, w, transpose_b=True) if ctx.needs_input_grad[0] else None
        grad_w = matmul_bf16(x, grad_preact, transpose_a=True) if ctx.needs_input_grad[1] else None
        return grad_x, grad_w


def _rows_of_gradient(g: torch.Tensor) -> torch.Tensor:
    """An incoming gradient as the kernels take it: dense rows, 16-byte aligned (a gradient may be
    a broadcast value or a slice that starts anywhere)."""
    g = g.contiguous()
    return g if g.data_ptr() % 16 == 0 else g.clone()


class FusedSwiGLUPreactFunction(torch.autograd.Function):
    """The same stage over saved pre-activations (8 bits or bf16) instead of the two factors.  The
    backward recomputes what it needs from them and leaves them as they are."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, w: torch.Tensor, checkpoint: str) -> torch.Tensor:
        h, pre = matmul_fused_swiglu_save_preact(x, w, checkpoint=checkpoint)
        ctx.save_for_backward(x, w, pre.data, pre.scales)
        ctx.bits, ctx.hidden = pre.bits, pre.hidden
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h: torch.Tensor):
        x, w, data, scales = ctx.saved_tensors
        grad_x, grad_w = fused_swiglu_backward_saved(
            x, w, _rows_of_gradient(grad_h), SavedPreact(data, scales, ctx.bits, ctx.hidden),
            need_x=ctx.needs_input_grad[0], need_w=ctx.needs_input_grad[1])
        return grad_x, grad_w, None


def fused_swiglu(x: torch.Tensor, w: torch.Tensor, *, checkpoint: str | None = None) -> torch.Tensor:
    """Differentiable ``silu(x @ W_gate) * (x @ W_up)`` with ``w = [W_up | W_gate]``.

    ``checkpoint`` says what the forward keeps for the backward besides its inputs: ``None`` two
    bf16 factors (``4N`` bytes per row), ``"bf16"`` the bf16 pre-activations (``4N``), ``"e4m3"`` the
    pre-activations in 8 bits (``2N + N/16``)."""
    if checkpoint is None:
        return FusedSwiGLUFunction.apply(x, w)
    _checkpoint_bits(checkpoint)
    return FusedSwiGLUPreactFunction.apply(x, w, checkpoint)


class FusedSwiGLUExpertsFunction(torch.autograd.Function):
    """The expert layer.  Kept for the backward: the inputs, the order, the pre-activations and,
    if the routing weights need a gradient, the experts' outputs.  The grouped copy of x and h
    are made again.

    Rounding to bf16 happens where a value becomes an operand of a product (h, the pre-activations'
    gradients) and once for each result; the experts' outputs and the rows of x's gradient, which
    are summed over a token's choices, stay in fp32, and the routing weight is applied to fp32
    values (``grouped_grad_preact``).  Each result then carries two roundings on its way."""

    @staticmethod
    def forward(ctx, x, expert_ids, weights, w, w_down, checkpoint):
        y, saved = experts_swiglu_save(x, expert_ids, weights, w, w_down, checkpoint=checkpoint)
        pre = saved.preact
        ctx.save_for_backward(x, weights, w, w_down, saved.order, pre.data, pre.scales,
                              saved.outputs if ctx.needs_input_grad[2] else None)
        ctx.bits, ctx.hidden = pre.bits, pre.hidden
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y: torch.Tensor):
        x, weights, w, w_down, order, data, scales, outputs = ctx.saved_tensors
        need_x, _, need_weights, need_w, need_down, _ = ctx.needs_input_grad
        saved = SavedExperts(order, SavedPreact(data, scales, ctx.bits, ctx.hidden), outputs)
        grad_x, grad_weights, grad_w, grad_down = experts_swiglu_backward(
            _rows_of_gradient(grad_y), x, weights, w, w_down, saved,
            need=(need_x, need_weights, need_w, need_down))
        return grad_x, None, grad_weights, grad_w, grad_down, None


def fused_swiglu_experts(x, expert_ids, weights, w, w_down, *, checkpoint: str = "bf16"):
    """Differentiable expert layer: ``experts_swiglu`` with gradients for ``x``, ``weights``, ``w``
    and ``w_down``.

    Kept for the backward, for each of the ``T * k`` slots: the pre-activations as ``checkpoint`` says
    (``"bf16"``: ``4N`` bytes, ``"e4m3"``: ``2N + N/16``) and, if ``weights`` needs a gradient, the experts'
    outputs in fp32 (``4 * D_out`` bytes, whatever the checkpoint).  With small experts the outputs are
    the larger part: at ``D_out = 2048``, ``N = 1024`` ``"e4m3"`` keeps 10.3 KB a slot, ``"bf16"`` 12.3."""
    return FusedSwiGLUExpertsFunction.apply(x, expert_ids, weights, w, w_down, checkpoint)
