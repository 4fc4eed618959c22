"""Mixture-of-experts operators around the SwiGLU stage.

A router gives every token ``k`` experts (``expert_ids[T, k]``) and weights (``weights[T, k]``);
expert ``e`` owns ``W[e] = [W_up | W_gate]`` (``[K, 2N]``) and ``W_down[e]`` (``[N, D]``).

``expert_order``          token slots sorted by expert (stable; ids outside ``[0, E)`` are dropped)
``expert_dispatch``       rows of ``x`` copied to their experts' row groups
``expert_combine``        rows summed back to tokens with the routing weights (without weights:
                          the gradient of ``expert_dispatch``)
``expert_combine_grad``   gradients of the weighted sum, for the rows and for the weights
``grouped_fused_swiglu``  the gate/up stage over row groups (``_save`` keeps the pre-activations)
``grouped_matmul``        the down projection over row groups, and its transposed form
``grouped_grad_preact``   the gate/up stage's backward behind the down projection, one launch
``grouped_weight_grad``   ``a_e^T @ g_e`` for every expert
``experts_swiglu``        all of the forward in one call, for inference
``experts_swiglu_save``   the same for training, and ``experts_swiglu_backward``, its backward
``swiglu_grad_preact_saved``  the backward's elementwise step from saved pre-activations
``fused_swiglu_backward_saved``  the dense stage's whole backward from them

The conventions are those of the other operators: bf16 tensors with unit column stride and 16-byte
rows, checks before anything is launched, torch's current stream unless ``stream=`` is given,
``out=`` for caller-owned results (which overlap no operand unless an operator allows it), no CPU
path.  The row counts of the groups live on the device
(``offsets``): no call here waits for the GPU.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib, tile_table
from .ops import (DTYPE, _check_matrix, _ld, _prep_out, _same_device, _stream_handle,
                  stream_context)

MAX_EXPERTS = 1024
MAX_CHOICES = 64
_ID_TYPES = (torch.int64, torch.int32)
_WEIGHT_TYPES = (torch.float32, torch.bfloat16)
_ONE_CTA_SLOTS = 2048      # up to here sgl_expert_order needs no scratch


class _launch:
    """``with _launch(stream, dev) as handle:`` makes ``dev`` the current device and ``stream``, if one
    is given, torch's current stream (so that allocations inside are ordered with the launch),
    and yields the raw stream handle.  Costs next to nothing where neither has to change."""

    __slots__ = ("stream", "dev", "prev", "ctx")

    def __init__(self, stream, dev: torch.device):
        self.stream = stream
        self.dev = dev
        self.prev = -1
        self.ctx = None

    def __enter__(self) -> int:
        cur = torch.cuda.current_device()
        if cur != self.dev.index:
            self.prev = cur
            torch.cuda.set_device(self.dev.index)
        if self.stream is not None:
            try:
                ctx = stream_context(self.stream, self.dev)
                ctx.__enter__()
            except BaseException:
                self.__exit__()
                raise
            self.ctx = ctx
        return _stream_handle(self.stream, self.dev)

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)
        if self.prev >= 0:
            torch.cuda.set_device(self.prev)
        return False


def _empty2(rows: int, cols: int, dtype, device) -> torch.Tensor:
    # (empty_strided parses its arguments about 1 us faster than empty with a shape)
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


class ExpertOrder(NamedTuple):
    """``offsets[E + 1]``: first row of every expert, then the number of kept slots;
    ``slots[T * k]``: the slot ``t * k + j`` each row holds (-1 behind ``offsets[E]``);
    ``rows[T, k]``: the row of each slot (-1 if dropped).  All int32, on the device."""

    offsets: torch.Tensor
    slots: torch.Tensor
    rows: torch.Tensor


class SavedPreact(NamedTuple):
    """Pre-activations ``[up | gate]`` kept for the backward pass.  ``data``: bf16 values
    (``bits == 16``) or e4m3 codes as uint8 (``bits == 8``), ``[rows, 2, padded columns]``;
    ``scales``: for 8 bits the exponents + 127 of the blocks of 32 columns,
    ``[rows, 2, blocks (even)]`` uint8.  ``hidden`` is the number of columns of either half."""

    data: torch.Tensor
    scales: torch.Tensor | None
    bits: int
    hidden: int


_CHECKPOINT_BITS = {"bf16": 16, "e4m3": 8}


def _checkpoint_bits(checkpoint: str) -> int:
    if checkpoint not in _CHECKPOINT_BITS:
        raise ValueError(f"checkpoint must be 'bf16' or 'e4m3', got {checkpoint!r}")
    return _CHECKPOINT_BITS[checkpoint]


def _check_choices(t: torch.Tensor, name: str, dtypes) -> None:
    """A [T, k] tensor of the router, any row pitch."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be [tokens, choices], got shape {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {', '.join(map(str, dtypes))}, got {t.dtype}")
    T, k = t.shape
    if not 1 <= k <= MAX_CHOICES:
        raise ValueError(f"{name} has {k} choices per token; 1 to {MAX_CHOICES} are supported")
    if k > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have unit stride along the choices, got {t.stride()}")
    if T > 1 and t.stride(0) < k:
        raise ValueError(f"{name} has overlapping rows: strides {t.stride()}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")


def _choice_ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_experts(w: torch.Tensor, name: str) -> None:
    if not isinstance(w, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(w).__name__}")
    if w.dim() != 3:
        raise ValueError(f"{name} must be [experts, rows, columns], got shape {tuple(w.shape)}")
    if w.dtype != DTYPE:
        raise TypeError(f"{name} must be torch.bfloat16, got {w.dtype}")
    if not w.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
    E, r, c = w.shape
    if not 1 <= E <= MAX_EXPERTS or r < 1 or c < 1:
        raise ValueError(f"{name} of shape {tuple(w.shape)}: 1 to {MAX_EXPERTS} experts with "
                         "non-empty matrices are supported")
    s0, s1, s2 = w.stride()
    if s2 != 1 or (r > 1 and (s1 < c or s1 % 8)):
        raise ValueError(f"{name} must be row-major with a row stride that is a multiple of 8, "
                         f"got strides {(s0, s1, s2)}")
    if E > 1 and (s0 % 8 or s0 < (r - 1) * s1 + c):
        raise ValueError(f"{name}: the experts' matrices overlap or are not 16-byte apart: strides "
                         f"{(s0, s1, s2)}")
    if w.data_ptr() % 16 != 0:
        raise ValueError(f"{name} must be 16-byte aligned")


def _expert_ld(w: torch.Tensor) -> int:
    return w.stride(1) if w.shape[1] > 1 else (w.shape[2] + 7) // 8 * 8


def _check_ints(t: torch.Tensor, name: str, shape: tuple) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be torch.int32, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_order_rows(order: ExpertOrder) -> tuple[int, int]:
    if not isinstance(order, ExpertOrder):
        raise TypeError(f"order must be an ExpertOrder, got {type(order).__name__}")
    if not isinstance(order.rows, torch.Tensor) or order.rows.dim() != 2:
        raise ValueError("order.rows must be a [tokens, choices] tensor")
    T, k = order.rows.shape
    _check_ints(order.rows, "order.rows", (T, k))
    if not 1 <= k <= MAX_CHOICES:
        raise ValueError(f"order.rows has {k} choices per token; 1 to {MAX_CHOICES} are supported")
    return T, k


def _check_rows(t: torch.Tensor, name: str) -> None:
    """Rows of the experts' outputs: a bf16 matrix as everywhere, or the same in fp32."""
    if isinstance(t, torch.Tensor) and t.dtype == torch.float32:
        if t.dim() != 2:
            raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
        rows, cols = t.shape
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
        if cols < 1 or t.stride(1) != 1 or (rows > 1 and (t.stride(0) < cols or t.stride(0) % 8)):
            raise ValueError(f"{name} must be row-major with a row stride that is a multiple of 8, "
                             f"got shape {tuple(t.shape)}, strides {t.stride()}")
        if t.data_ptr() % 16 != 0:
            raise ValueError(f"{name} must be 16-byte aligned")
        return
    _check_matrix(t, name, allow_empty_rows=True)


def _prep_rows(out, M: int, N: int, device, dtype=DTYPE):
    """``out`` for a result in ``dtype`` (bf16 or fp32), allocated if omitted."""
    if out is None:
        return _empty2(M, N, dtype, device)
    if dtype == DTYPE:
        return _prep_out(out, M, N, device)
    if not isinstance(out, torch.Tensor) or out.dtype != dtype:
        raise TypeError(f"out must be a {dtype} tensor")
    _check_rows(out, "out")
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out shape {tuple(out.shape)} != {(M, N)}")
    if out.device != device:
        raise ValueError(f"out is on {out.device}, expected {device}")
    return out


# Plain operands are recognised with a few attribute reads (the calls below cost microseconds, the
# small problems they are for not many more); anything else goes through the full checks, which say
# what is wrong or accept it with its strides.


def _matrix(t, name: str) -> tuple[int, int, int]:
    """Checks a bf16 matrix (rows may be none); (rows, columns, row pitch)."""
    if type(t) is torch.Tensor and t.dtype is DTYPE and t.is_cuda and t.dim() == 2 \
            and t.is_contiguous():
        rows, cols = t.shape
        if cols and cols % 8 == 0 and t.data_ptr() % 16 == 0:
            return rows, cols, cols
    _check_matrix(t, name, allow_empty_rows=True)
    return t.shape[0], t.shape[1], _ld(t)


def _rows_matrix(t, name: str) -> tuple[int, int, int]:
    """The same for rows that may be fp32."""
    if isinstance(t, torch.Tensor) and t.dtype is torch.float32:
        _check_rows(t, name)
        return t.shape[0], t.shape[1], _ld(t)
    return _matrix(t, name)


def _order_rows(order) -> tuple[int, int]:
    """Checks an order's ``rows``; (tokens, choices)."""
    if type(order) is ExpertOrder:
        rows = order.rows
        if type(rows) is torch.Tensor and rows.dtype is torch.int32 and rows.is_cuda \
                and rows.dim() == 2 and rows.is_contiguous():
            T, k = rows.shape
            if 0 < k <= MAX_CHOICES:
                return T, k
    return _check_order_rows(order)


def _choices(t, name: str, dtypes) -> tuple[int, int, int]:
    """Checks a router's [T, k] tensor; (tokens, choices, row pitch)."""
    if type(t) is torch.Tensor and t.dtype in dtypes and t.is_cuda and t.dim() == 2 \
            and t.is_contiguous():
        T, k = t.shape
        if 0 < k <= MAX_CHOICES:
            return T, k, k
    _check_choices(t, name, dtypes)
    return t.shape[0], t.shape[1], _choice_ld(t)


def _weights(weights, T: int, k: int) -> int:
    """Checks routing weights; their row pitch."""
    T2, k2, ld = _choices(weights, "weights", _WEIGHT_TYPES)
    if T2 != T or k2 != k:
        raise ValueError(f"weights shape {(T2, k2)} != {(T, k)}")
    return ld


def _one_device(*tensors) -> torch.device:
    """The device of all of them."""
    first = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != first:
            raise ValueError("operands are on different devices: "
                             + ", ".join(str(u.device) for u in tensors))
    return tensors[0].device


def _multiple_of_8(**sizes: int) -> None:
    for name, n in sizes.items():
        if n % 8:
            raise ValueError(f"{name}={n} must be a multiple of 8")


def expert_order(expert_ids, num_experts: int, *, stream=None) -> ExpertOrder:
    """Sorts the slots of ``expert_ids[T, k]`` (int32 or int64) by expert, slot order kept inside
    an expert.  Slots with an id outside ``[0, num_experts)`` are dropped."""
    T, k, ld = _choices(expert_ids, "expert_ids", _ID_TYPES)
    E = int(num_experts)
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"num_experts={E} outside [1, {MAX_EXPERTS}]")
    dev = expert_ids.device
    R = T * k
    with _launch(stream, dev) as handle:
        offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
        slots = torch.empty(R, dtype=torch.int32, device=dev)
        rows = _empty2(T, k, torch.int32, dev)
        if T == 0:
            offsets.zero_()
            return ExpertOrder(offsets, slots, rows)
        lib = _lib.load()
        need, scratch = 0, None
        if R > _ONE_CTA_SLOTS:
            need = lib.sgl_expert_order_scratch_bytes(T, k, E)
            scratch = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        _lib.check(lib.sgl_expert_order(
            expert_ids.data_ptr(), expert_ids.dtype is torch.int64, T, k, ld, E,
            offsets.data_ptr(), slots.data_ptr(), rows.data_ptr(),
            scratch.data_ptr() if scratch is not None else None, need, handle))
    return ExpertOrder(offsets, slots, rows)


def expert_dispatch(x, order: ExpertOrder, *, out=None, stream=None):
    """``out[order.rows[t, j]] = x[t]``: ``[T, D]`` -> ``[T * k, D]``, rows grouped by expert.  Rows
    behind the last expert's (there are some if slots were dropped) are left as they were."""
    T, k = _order_rows(order)
    T2, D, ldx = _matrix(x, "x")
    if T2 != T:
        raise ValueError(f"x has {T2} rows, the order {T} tokens")
    _multiple_of_8(D=D)
    dev = _one_device(x, order.rows)
    if T == 0:
        return out if out is not None else torch.empty((0, D), dtype=DTYPE, device=dev)
    with _launch(stream, dev) as handle:
        o = _prep_rows(out, T * k, D, dev)
        _lib.check(_lib.load().sgl_expert_dispatch(
            x.data_ptr(), order.rows.data_ptr(), o.data_ptr(), T, k, D, T * k, ldx, _ld(o), handle))
    return o


def expert_combine(rows, order: ExpertOrder, weights=None, *, out=None, stream=None):
    """``out[t] = sum_j weights[t, j] * rows[order.rows[t, j]]``: ``[T * k, D]`` bf16 or fp32 ->
    ``[T, D]`` bf16, fp32 sums in the order of ``j``.  ``weights`` is fp32 or bf16 ``[T, k]``;
    without weights the rows are summed as they are.  Dropped slots add nothing."""
    T, k = _order_rows(order)
    R, D, ld = _rows_matrix(rows, "rows")
    if R != T * k:
        raise ValueError(f"rows has {R} rows, the order {T * k} slots")
    _multiple_of_8(D=D)
    if weights is not None:
        ldw, w_ptr, w_bf16 = _weights(weights, T, k), weights.data_ptr(), weights.dtype is DTYPE
        dev = _one_device(rows, order.rows, weights)
    else:
        ldw, w_ptr, w_bf16 = 0, None, False
        dev = _one_device(rows, order.rows)
    if T == 0:
        return out if out is not None else torch.empty((0, D), dtype=DTYPE, device=dev)
    with _launch(stream, dev) as handle:
        o = _prep_rows(out, T, D, dev)
        _lib.check(_lib.load().sgl_expert_combine(
            rows.data_ptr(), rows.dtype is torch.float32, order.rows.data_ptr(), w_ptr, w_bf16,
            o.data_ptr(), T, k, D, R, ld, ldw, _ld(o), handle))
    return o


def expert_combine_grad(grad_out, rows, order: ExpertOrder, weights, *, weighted: bool = True,
                        out=None, stream=None):
    """Gradients of ``expert_combine(rows, order, weights)``: ``(grad_rows, grad_weights)`` with
    ``grad_rows[r] = weight * grad_out[t]`` (rows behind the last expert's are left as they were)
    and ``grad_weights[t, j] = <grad_out[t], rows[r]>`` in the weights' type, 0 for dropped slots.
    ``rows`` may be bf16 or fp32.  ``out`` takes ``grad_rows``; it may be a bf16 ``rows`` itself.
    With ``rows=None`` only ``grad_rows`` is computed (``grad_weights`` is None).  With
    ``weighted=False`` the rows of ``grad_rows`` are ``grad_out[t]`` as it is, for a caller that
    applies the weight further on (``grouped_grad_preact`` does)."""
    T, k = _order_rows(order)
    T2, D, ldg = _matrix(grad_out, "grad_out")
    R = T * k
    fits = T2 == T
    ld = D
    if rows is not None:
        R2, D2, ld = _rows_matrix(rows, "rows")
        fits = fits and R2 == R and D2 == D
    if not fits:
        raise ValueError(f"grad_out {tuple(grad_out.shape)} and rows "
                         f"{tuple(rows.shape) if rows is not None else None} do not fit {T} tokens "
                         f"of {k} choices")
    _multiple_of_8(D=D)
    ldw = _weights(weights, T, k)
    if rows is not None:
        dev = _one_device(grad_out, order.rows, weights, rows)
    else:
        dev = _one_device(grad_out, order.rows, weights)
    with _launch(stream, dev) as handle:
        gw = _empty2(T, k, weights.dtype, dev) if rows is not None else None
        if T == 0:
            return out if out is not None else torch.empty((0, D), dtype=DTYPE, device=dev), gw
        gr = _prep_rows(out, R, D, dev)
        _lib.check(_lib.load().sgl_expert_combine_grad(
            grad_out.data_ptr(), rows.data_ptr() if rows is not None else None,
            rows is not None and rows.dtype is torch.float32, order.rows.data_ptr(),
            weights.data_ptr() if weighted else None, weights.dtype is DTYPE, gr.data_ptr(),
            gw.data_ptr() if gw is not None else None, T, k, D, R, ldg, ld, ldw, _ld(gr), handle))
    return gr, gw


def _swiglu_operands(x, W, offsets):
    """Checks and sizes of the grouped gate/up stage: (R, K, N, E, device)."""
    _check_matrix(x, "x", allow_empty_rows=True)
    _check_experts(W, "W")
    R, K = x.shape
    E, K2, N2 = W.shape
    if K2 != K:
        raise ValueError(f"K mismatch: x.K={K} vs W.K={K2}")
    if N2 % 2:
        raise ValueError(f"W's last dim ({N2}) must be even")
    _multiple_of_8(K=K, N=N2 // 2)
    _check_ints(offsets, "offsets", (E + 1,))
    return R, K, N2 // 2, E, _same_device(("x", x), ("W", W), ("offsets", offsets))


def grouped_fused_swiglu(x, W, offsets, *, out=None, stream=None):
    """``h[r] = silu(x[r] @ W_gate[e]) * (x[r] @ W_up[e])`` for the rows ``[offsets[e],
    offsets[e + 1])`` of every expert.

    x       : [R, K] bf16
    W       : [E, K, 2N] bf16, ``[W_up | W_gate]`` per expert
    offsets : [E + 1] int32 on the device, non-decreasing
    returns : [R, N] bf16; rows behind ``offsets[E]`` are left as they were
    """
    R, K, N, E, dev = _swiglu_operands(x, W, offsets)
    if R == 0:
        return out if out is not None else torch.empty((0, N), dtype=DTYPE, device=dev)
    with _launch(stream, dev) as handle:
        h = _prep_rows(out, R, N, dev)
        _lib.check(_lib.load().sgl_grouped_fused_swiglu(
            x.data_ptr(), W.data_ptr(), offsets.data_ptr(), h.data_ptr(), R, N, K, E, _ld(x),
            _expert_ld(W), W.stride(0), _ld(h), handle))
    return h


def _preact_shapes(bits: int, rows: int, N: int):
    """Shapes of ``SavedPreact.data`` and ``.scales`` (None for 16 bits): halves padded to whole
    blocks of 32 columns, an even number of scales (``sgl_preact_bytes`` has the same in bytes)."""
    return (rows, 2, (N + 31) // 32 * 32), (rows, 2, (N + 63) // 64 * 2) if bits == 8 else None


def _empty_preact(bits: int, rows: int, N: int, dev) -> SavedPreact:
    shape, scale_shape = _preact_shapes(bits, rows, N)
    data = torch.empty(shape, dtype=torch.uint8 if bits == 8 else DTYPE, device=dev)
    scales = torch.empty(scale_shape, dtype=torch.uint8, device=dev) if bits == 8 else None
    return SavedPreact(data, scales, bits, N)


def _check_preact(p: SavedPreact) -> None:
    if not isinstance(p, SavedPreact):
        raise TypeError(f"preact must be a SavedPreact, got {type(p).__name__}")
    if not isinstance(p.data, torch.Tensor) or p.data.dim() != 3:
        raise ValueError("preact.data must be a [rows, 2, columns] tensor")
    if p.bits not in (8, 16):
        raise ValueError(f"preact.bits must be 8 or 16, got {p.bits}")
    shape, scale_shape = _preact_shapes(p.bits, p.data.shape[0], p.hidden)
    for name, t, want, dtype in (("data", p.data, shape, torch.uint8 if p.bits == 8 else DTYPE),
                                 ("scales", p.scales, scale_shape, torch.uint8)):
        if want is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != want \
                or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"preact.{name} must be a contiguous {dtype} CUDA tensor of shape {want}")


def _save(x, w_ptr, offsets, E, ldx, ldw, w_stride, R, K, N, bits, out, stream, dev):
    with _launch(stream, dev) as handle:
        h = _prep_rows(out, R, N, dev) if R else torch.empty((0, N), dtype=DTYPE, device=dev)
        pre = _empty_preact(bits, R, N, dev)
        if R:
            _lib.check(_lib.load().sgl_grouped_fused_swiglu_save(
                x.data_ptr(), w_ptr, offsets.data_ptr() if offsets is not None else None,
                h.data_ptr(), pre.data.data_ptr(),
                pre.scales.data_ptr() if pre.scales is not None else None, bits, R, N, K, E, ldx,
                ldw, w_stride, _ld(h), handle))
    return h, pre


def grouped_fused_swiglu_save(x, W, offsets, *, checkpoint: str = "bf16", out=None, stream=None):
    """Training form of ``grouped_fused_swiglu``: ``(h, SavedPreact)``.  ``checkpoint="e4m3"`` keeps
    the pre-activations in 8 bits (a power-of-two scale per row and 32 columns), ``"bf16"`` in 16."""
    bits = _checkpoint_bits(checkpoint)
    R, K, N, E, dev = _swiglu_operands(x, W, offsets)
    return _save(x, W.data_ptr(), offsets, E, _ld(x), _expert_ld(W), W.stride(0), R, K, N, bits, out,
                 stream, dev)


def matmul_fused_swiglu_save_preact(A, W, *, checkpoint: str = "e4m3", out=None, stream=None):
    """``matmul_fused_swiglu`` for training with an 8-bit checkpoint: ``(h, SavedPreact)``.

    A : [M, K] bf16, W : [K, 2N] bf16 = [W_up | W_gate].  The checkpoint takes ``2N + N/16`` bytes
    per row (``"bf16"``: ``4N``); ``matmul_fused_swiglu_save_factors`` keeps two bf16 factors."""
    bits = _checkpoint_bits(checkpoint)
    M, K, ldx, N, ldw, dev = _stage_operands(A, W)
    return _save(A, W.data_ptr(), None, 1, ldx, ldw, 0, M, K, N, bits, out, stream, dev)


def _stage_operands(A, W):
    """Checks and sizes of the dense stage: (M, K, pitch of A, N, pitch of W, device)."""
    M, K, ldx = _matrix(A, "A")
    K2, N2, ldw = _matrix(W, "W")
    if K != K2 or K == 0:
        raise ValueError(f"K mismatch: A.K={K} vs W.K={K2}")
    if N2 % 2:
        raise ValueError(f"W's 2nd dim ({N2}) must be even")
    _multiple_of_8(K=K, N=N2 // 2)
    return M, K, ldx, N2 // 2, ldw, _one_device(A, W)


def fused_swiglu_backward_saved(x, W, dy, preact: SavedPreact, *, need_x: bool = True,
                                need_w: bool = True, stream=None):
    """The dense stage's backward from saved pre-activations, one library call: ``(grad_x [M, K],
    grad_w [K, 2N])`` for ``h = matmul_fused_swiglu(x, W)`` and its gradient ``dy [M, N]``; None for
    the one that is not needed.  The two products are ``matmul_bf16``'s, tile table included."""
    M, K, ldx, N, ldw, dev = _stage_operands(x, W)
    M2, N2, lddy = _matrix(dy, "dy")
    _check_preact(preact)
    if M2 != M or N2 != N or preact.hidden != N or preact.data.shape[0] != M:
        raise ValueError(f"dy shape {tuple(dy.shape)} or the saved pre-activations of "
                         f"{preact.data.shape[0]} rows and {preact.hidden} columns do not fit x "
                         f"{tuple(x.shape)} and W {tuple(W.shape)}")
    _one_device(x, dy, preact.data, *(() if preact.scales is None else (preact.scales,)))
    with _launch(stream, dev) as handle:
        gx = _empty2(M, K, DTYPE, dev) if need_x else None
        gw = _empty2(K, 2 * N, DTYPE, dev) if need_w else None
        if M == 0:
            return gx, gw.zero_() if need_w else None
        gp = _empty2(M, 2 * N, DTYPE, dev)
        cfg_x = tile_table.lookup(_lib.FORM_MATMUL, M, K, 2 * N)
        cfg_w = tile_table.lookup(_lib.FORM_MATMUL, K, 2 * N, M)
        _lib.check(_lib.load().sgl_fused_swiglu_backward_saved(
            x.data_ptr(), W.data_ptr(), dy.data_ptr(), preact.data.data_ptr(),
            preact.scales.data_ptr() if preact.scales is not None else None, preact.bits,
            gp.data_ptr(), gx.data_ptr() if need_x else None, gw.data_ptr() if need_w else None,
            M, N, K, ldx, ldw, lddy, C.byref(cfg_x.to_c()) if cfg_x is not None else None,
            C.byref(cfg_w.to_c()) if cfg_w is not None else None, handle))
    return gx, gw


def swiglu_grad_preact_saved(dy, preact: SavedPreact, *, offsets=None, return_h: bool = False,
                             out=None, stream=None):
    """Backward elementwise step from saved pre-activations: ``[dy * silu(gate) |
    dy * up * silu'(gate)]``, ``[R, 2N]``; with ``return_h`` also ``h = silu(gate) * up``.  With
    ``offsets`` (of the experts' row groups) rows behind ``offsets[-1]`` are left as they were."""
    _check_preact(preact)
    R, N, lddy = _matrix(dy, "dy")
    _multiple_of_8(N=N)
    if preact.hidden != N or preact.data.shape[0] != R:
        raise ValueError(f"dy shape {tuple(dy.shape)} does not fit the saved pre-activations of "
                         f"{preact.data.shape[0]} rows and {preact.hidden} columns")
    named = [("dy", dy), ("preact.data", preact.data)]
    if preact.scales is not None:
        named.append(("preact.scales", preact.scales))
    if offsets is not None:
        if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must be a 1-D tensor")
        _check_ints(offsets, "offsets", (offsets.numel(),))
        named.append(("offsets", offsets))
    dev = _same_device(*named)
    end = offsets.data_ptr() + 4 * (offsets.numel() - 1) if offsets is not None else None
    with _launch(stream, dev) as handle:
        h = _empty2(R, N, DTYPE, dev) if return_h else None
        if R == 0:
            g = out if out is not None else torch.empty((0, 2 * N), dtype=DTYPE, device=dev)
            return (g, h) if return_h else g
        g = _prep_rows(out, R, 2 * N, dev)
        _lib.check(_lib.load().sgl_swiglu_grad_preact_saved(
            dy.data_ptr(), preact.data.data_ptr(),
            preact.scales.data_ptr() if preact.scales is not None else None, preact.bits,
            g.data_ptr(), h.data_ptr() if h is not None else None, end, R, N, lddy, _ld(g),
            _ld(h) if h is not None else 0, handle))
    return (g, h) if return_h else g


def grouped_matmul(a, B, offsets, *, out=None, stream=None, transpose_b: bool = False,
                   out_dtype: torch.dtype = DTYPE):
    """``c[r] = a[r] @ B[e]`` for the rows of every expert: the down projection.

    a : [R, K] bf16;  B : [E, K, N] bf16, or [E, N, K] with ``transpose_b`` (read in place)
    returns [R, N] in ``out_dtype``, bf16 or fp32; rows behind ``offsets[E]`` are left as they were
    """
    if out_dtype not in (DTYPE, torch.float32):
        raise TypeError(f"out_dtype must be torch.bfloat16 or torch.float32, got {out_dtype}")
    _check_matrix(a, "a", allow_empty_rows=True)
    _check_experts(B, "B")
    R, K = a.shape
    E = B.shape[0]
    K2, N = (B.shape[2], B.shape[1]) if transpose_b else (B.shape[1], B.shape[2])
    if K2 != K:
        raise ValueError(f"K mismatch: a.K={K} vs op(B).K={K2}")
    _multiple_of_8(K=K, N=N)
    _check_ints(offsets, "offsets", (E + 1,))
    dev = _same_device(("a", a), ("B", B), ("offsets", offsets))
    if R == 0:
        return out if out is not None else torch.empty((0, N), dtype=out_dtype, device=dev)
    with _launch(stream, dev) as handle:
        c = _prep_rows(out, R, N, dev, out_dtype)
        _lib.check(_lib.load().sgl_grouped_matmul(
            a.data_ptr(), B.data_ptr(), offsets.data_ptr(), c.data_ptr(), R, N, K, E, _ld(a),
            _expert_ld(B), B.stride(0), _ld(c), int(transpose_b), int(out_dtype == torch.float32),
            handle))
    return c


def grouped_grad_preact(grad_rows, W_down, preact: SavedPreact, order: ExpertOrder, weights=None, *,
                        out=None, stream=None):
    """The gate/up stage's backward behind the down projection, one launch: with
    ``t = grad_rows[r] @ W_down[e]^T`` and the saved pre-activations of row ``r``,
    ``grad_preact[r] = [w t silu(gate) | w t up silu'(gate)]`` and ``h[r] = w silu(gate) up``, ``w`` the
    routing weight of the row's slot (1 without ``weights``).  ``t`` is not rounded; ``W_down``'s
    gradient is ``grouped_weight_grad(h, grad_rows, offsets)``, the weight being in ``h`` already.

    grad_rows : [R, D] bf16, gradients of the rows' outputs without the routing weight
    W_down    : [E, N, D] bf16
    returns   : ``(grad_preact [R, 2N], h [R, N])``; rows behind the last expert's are left as they were
    """
    T, k = _order_rows(order)
    _check_matrix(grad_rows, "grad_rows", allow_empty_rows=True)
    _check_experts(W_down, "W_down")
    R, D = grad_rows.shape
    E, N, D2 = W_down.shape
    if D2 != D or R != T * k:
        raise ValueError(f"grad_rows {tuple(grad_rows.shape)} does not fit W_down "
                         f"{tuple(W_down.shape)} and {T} tokens of {k} choices")
    _multiple_of_8(D=D, N=N)
    _check_preact(preact)
    if preact.hidden != N or preact.data.shape[0] != R:
        raise ValueError(f"the saved pre-activations are of {preact.data.shape[0]} rows and "
                         f"{preact.hidden} columns, expected {R} and {N}")
    _check_ints(order.offsets, "order.offsets", (E + 1,))
    _check_ints(order.slots, "order.slots", (R,))
    named = [("grad_rows", grad_rows), ("W_down", W_down), ("preact.data", preact.data),
             ("order.rows", order.rows), ("order.offsets", order.offsets),
             ("order.slots", order.slots)]
    if preact.scales is not None:
        named.append(("preact.scales", preact.scales))
    ldw = 0
    if weights is not None:
        ldw = _weights(weights, T, k)
        named.append(("weights", weights))
    dev = _same_device(*named)
    with _launch(stream, dev) as handle:
        h = _empty2(R, N, DTYPE, dev)
        if R == 0:
            return (out if out is not None else torch.empty((0, 2 * N), dtype=DTYPE, device=dev)), h
        g = _prep_rows(out, R, 2 * N, dev)
        _lib.check(_lib.load().sgl_grouped_grad_preact(
            grad_rows.data_ptr(), W_down.data_ptr(), order.offsets.data_ptr(),
            order.slots.data_ptr() if weights is not None else None,
            weights.data_ptr() if weights is not None else None,
            int(weights is not None and weights.dtype == DTYPE), preact.data.data_ptr(),
            preact.scales.data_ptr() if preact.scales is not None else None, preact.bits,
            g.data_ptr(), h.data_ptr(), R, N, D, E, k, _ld(grad_rows), _expert_ld(W_down),
            W_down.stride(0), ldw, _ld(g), _ld(h), handle))
    return g, h


def grouped_weight_grad(a, g, offsets, *, out=None, stream=None):
    """``C[e] = a_e^T @ g_e`` over the rows of every expert: ``a [R, M]``, ``g [R, N]`` ->
    ``[E, M, N]`` bf16 (fp32 sums; zero for an expert without rows)."""
    _check_matrix(a, "a", allow_empty_rows=True)
    _check_matrix(g, "g", allow_empty_rows=True)
    R, M = a.shape
    if g.shape[0] != R:
        raise ValueError(f"a has {R} rows, g {g.shape[0]}")
    N = g.shape[1]
    _multiple_of_8(M=M, N=N)
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or \
            not 2 <= offsets.numel() <= MAX_EXPERTS + 1:
        raise ValueError(f"offsets must be a 1-D tensor of 2 to {MAX_EXPERTS + 1} entries")
    E = offsets.numel() - 1
    _check_ints(offsets, "offsets", (E + 1,))
    dev = _same_device(("a", a), ("g", g), ("offsets", offsets))
    with _launch(stream, dev) as handle:
        if out is None:
            c = torch.empty((E, M, N), dtype=DTYPE, device=dev)
        else:
            c = out
            _check_experts(c, "out")
            if tuple(c.shape) != (E, M, N):
                raise ValueError(f"out shape {tuple(c.shape)} != {(E, M, N)}")
            if c.device != dev:
                raise ValueError(f"out is on {c.device}, expected {dev}")
        if R == 0:
            return c.zero_()
        _lib.check(_lib.load().sgl_grouped_weight_grad(
            a.data_ptr(), g.data_ptr(), offsets.data_ptr(), c.data_ptr(), R, M, N, E, _ld(a), _ld(g),
            _expert_ld(c), c.stride(0), handle))
    return c


def experts_swiglu_workspace_bytes(T: int, k: int, E: int, D: int, N: int, D_out: int) -> int:
    """Bytes of device memory ``experts_swiglu`` works in for these sizes."""
    n = _lib.load().sgl_experts_swiglu_workspace_bytes(T, k, E, D, N, D_out)
    if n < 0:
        _lib.check(int(n))
    return int(n)


def _layer_operands(x, expert_ids, weights, W, W_down):
    """Checks and sizes of the expert layer: (T, k, E, D, N, D_out, pitches of x, ids and weights,
    device)."""
    T, D, ldx = _matrix(x, "x")
    T2, k, ld_ids = _choices(expert_ids, "expert_ids", _ID_TYPES)
    if T2 != T:
        raise ValueError(f"x has {T} rows, expert_ids {T2}")
    ldw = _weights(weights, T, k)
    _check_experts(W, "W")
    _check_experts(W_down, "W_down")
    E, D2, N2 = W.shape
    if D2 != D:
        raise ValueError(f"K mismatch: x.K={D} vs W.K={D2}")
    if N2 % 2:
        raise ValueError(f"W's last dim ({N2}) must be even")
    N = N2 // 2
    E2, N3, D_out = W_down.shape
    if E2 != E or N3 != N:
        raise ValueError(f"W_down shape {tuple(W_down.shape)} does not follow W's {tuple(W.shape)}")
    _multiple_of_8(K=D, N=N, D=D_out)
    return (T, k, E, D, N, D_out, ldx, ld_ids, ldw,
            _one_device(x, expert_ids, weights, W, W_down))


def experts_swiglu(x, expert_ids, weights, W, W_down, *, out=None, workspace=None, stream=None):
    """The expert layer at inference, one library call:
    ``y[t] = sum_j weights[t, j] * (silu(x[t] @ W_gate[e]) * (x[t] @ W_up[e])) @ W_down[e]`` with
    ``e = expert_ids[t, j]``.  The activation's result is rounded to bf16, the down projection's operand
    type; everything else on the way to ``y`` stays in fp32.

    x          : [T, D] bf16
    expert_ids : [T, k] int32 or int64; a slot outside ``[0, E)`` is dropped
    weights    : [T, k] fp32 or bf16
    W, W_down  : [E, D, 2N] = [W_up | W_gate], [E, N, D_out] bf16
    workspace  : uint8 CUDA tensor of ``experts_swiglu_workspace_bytes`` bytes (allocated if omitted);
                 calls that overlap on the GPU must not share one
    returns    : [T, D_out] bf16
    """
    T, k, E, D, N, D_out, ldx, ld_ids, ldw, dev = _layer_operands(x, expert_ids, weights, W, W_down)
    if T == 0:
        return out if out is not None else torch.empty((0, D_out), dtype=DTYPE, device=dev)
    lib = _lib.load()
    need = lib.sgl_experts_swiglu_workspace_bytes(T, k, E, D, N, D_out)
    if need < 0:
        _lib.check(int(need))
    with _launch(stream, dev) as handle:
        y = _prep_rows(out, T, D_out, dev)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        elif workspace.dtype != torch.uint8 or workspace.device != dev \
                or not workspace.is_contiguous():
            raise ValueError(
                "workspace must be a contiguous uint8 CUDA tensor on the operands' device")
        _lib.check(lib.sgl_experts_swiglu(
            x.data_ptr(), expert_ids.data_ptr(), expert_ids.dtype is torch.int64,
            weights.data_ptr(), weights.dtype is DTYPE, W.data_ptr(), W_down.data_ptr(),
            y.data_ptr(), workspace.data_ptr(), workspace.numel(), T, k, E, D, N, D_out, ldx, ld_ids,
            ldw, _expert_ld(W), W.stride(0), _expert_ld(W_down), W_down.stride(0), _ld(y), handle))
    return y


class SavedExperts(NamedTuple):
    """What ``experts_swiglu_save`` keeps for the backward: the order as one int32 tensor (offsets,
    slots, rows), the pre-activations, the experts' outputs ``[T * k, D_out]`` in fp32."""

    order: torch.Tensor
    preact: SavedPreact
    outputs: torch.Tensor


def experts_swiglu_save(x, expert_ids, weights, W, W_down, *, checkpoint: str = "bf16", stream=None):
    """The expert layer for training, one library call: ``(y [T, D_out], SavedExperts)``.  Operands as
    for ``experts_swiglu``; ``checkpoint`` as for ``grouped_fused_swiglu_save``.  ``outputs`` takes
    ``4 * D_out`` bytes a slot beside the checkpoint; drop it if ``weights`` needs no gradient."""
    bits = _checkpoint_bits(checkpoint)
    T, k, E, D, N, D_out, ldx, ld_ids, ldw, dev = _layer_operands(x, expert_ids, weights, W, W_down)
    R = T * k
    lib = _lib.load()
    with _launch(stream, dev) as handle:
        y = _empty2(T, D_out, DTYPE, dev)
        order = torch.empty(E + 1 + 2 * R, dtype=torch.int32, device=dev)
        pre = _empty_preact(bits, R, N, dev)
        ys = _empty2(R, D_out, torch.float32, dev)
        if T == 0:
            order.zero_()
            return y, SavedExperts(order, pre, ys)
        need = lib.sgl_experts_swiglu_train_workspace_bytes(T, k, E, D, N, D_out, 0)
        if need < 0:
            _lib.check(int(need))
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(lib.sgl_experts_swiglu_save(
            x.data_ptr(), expert_ids.data_ptr(), expert_ids.dtype is torch.int64,
            weights.data_ptr(), weights.dtype is DTYPE, W.data_ptr(), W_down.data_ptr(),
            y.data_ptr(), order.data_ptr(), pre.data.data_ptr(),
            pre.scales.data_ptr() if pre.scales is not None else None, bits, ys.data_ptr(),
            ws.data_ptr(), need, T, k, E, D, N, D_out, ldx, ld_ids, ldw, _expert_ld(W), W.stride(0),
            _expert_ld(W_down), W_down.stride(0), handle))
    return y, SavedExperts(order, pre, ys)


def experts_swiglu_backward(grad_y, x, weights, W, W_down, saved: SavedExperts, *,
                            need=(True, True, True, True), stream=None):
    """Backward of ``experts_swiglu_save``, one library call: gradients of ``x``, ``weights``, ``W`` and
    ``W_down``, None where ``need`` says so.  ``saved.outputs`` may be None if the weights need none."""
    T, D, ldx = _matrix(x, "x")
    T2, D_out, ldg = _matrix(grad_y, "grad_y")
    if not isinstance(saved, SavedExperts):
        raise TypeError(f"saved must be a SavedExperts, got {type(saved).__name__}")
    k = weights.shape[1] if isinstance(weights, torch.Tensor) and weights.dim() == 2 else 0
    ldw = _weights(weights, T, k)
    _check_experts(W, "W")
    _check_experts(W_down, "W_down")
    E, D2, N2 = W.shape
    N, R = N2 // 2, T * k
    if T2 != T or D2 != D or N2 % 2 or tuple(W_down.shape) != (E, N, D_out):
        raise ValueError(f"grad_y {tuple(grad_y.shape)}, x {tuple(x.shape)}, W {tuple(W.shape)} and "
                         f"W_down {tuple(W_down.shape)} do not belong together")
    _multiple_of_8(K=D, N=N, D=D_out)
    if ldg != D_out:
        raise ValueError(f"grad_y must be dense, got strides {grad_y.stride()}")
    order, pre, ys = saved
    _check_ints(order, "saved.order", (E + 1 + 2 * R,))
    _check_preact(pre)
    if pre.hidden != N or pre.data.shape[0] != R:
        raise ValueError(f"the saved pre-activations are of {pre.data.shape[0]} rows and {pre.hidden} "
                         f"columns, expected {R} and {N}")
    need_x, need_weights, need_w, need_down = need
    tensors = [x, grad_y, weights, W, W_down, order, pre.data]
    if pre.scales is not None:
        tensors.append(pre.scales)
    if need_weights:
        if ys is None:
            raise ValueError("saved.outputs is needed for the weights' gradient")
        R2, D3, ld_ys = _rows_matrix(ys, "saved.outputs")
        if ys.dtype is not torch.float32 or (R2, D3, ld_ys) != (R, D_out, D_out):
            raise ValueError(f"saved.outputs must be dense fp32 of shape {(R, D_out)}")
        tensors.append(ys)
    dev = _one_device(*tensors)
    lib = _lib.load()
    with _launch(stream, dev) as handle:
        gx = _empty2(T, D, DTYPE, dev) if need_x else None
        gr = _empty2(T, k, weights.dtype, dev) if need_weights else None
        gw = torch.empty((E, D, N2), dtype=DTYPE, device=dev) if need_w else None
        gd = torch.empty((E, N, D_out), dtype=DTYPE, device=dev) if need_down else None
        if T == 0:
            return gx, gr, gw.zero_() if need_w else None, gd.zero_() if need_down else None
        size = lib.sgl_experts_swiglu_train_workspace_bytes(T, k, E, D, N, D_out, 1)
        if size < 0:
            _lib.check(int(size))
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _lib.check(lib.sgl_experts_swiglu_backward(
            grad_y.data_ptr(), x.data_ptr(), weights.data_ptr(), weights.dtype is DTYPE,
            W.data_ptr(), W_down.data_ptr(), order.data_ptr(), pre.data.data_ptr(),
            pre.scales.data_ptr() if pre.scales is not None else None, pre.bits,
            ys.data_ptr() if need_weights else None, gx.data_ptr() if need_x else None,
            gr.data_ptr() if need_weights else None, gw.data_ptr() if need_w else None,
            gd.data_ptr() if need_down else None, ws.data_ptr(), size, T, k, E, D, N, D_out, ldx,
            ldw, _expert_ld(W), W.stride(0), _expert_ld(W_down), W_down.stride(0), handle))
    return gx, gr, gw, gd
