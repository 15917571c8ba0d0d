"""Tokens sorted by expert and back, with routing weights, and the gradients of both.

``quantize_group_rows`` and ``combine_rows`` serve a forward pass on quantised rows; the functions
here move bf16, fp16 and fp32 rows, keep the plan that leads back, and are differentiable: the way
there and back of an expert layer that is trained, or served in 16 bits.  The layouts are the ones
the grouped GEMMs read: ``align=128`` (or 256) with ``plan.m_indices`` for the contiguous entry
points, ``align=1`` with ``plan.counts`` / ``plan.offsets`` for the compact one.  CUDA tensors only.

Rows that stand for no pair (an expert's padding, everything behind the last expert;
``plan.m_indices < 0``) are zero in what these functions allocate and are left as they are in a
buffer that the caller passes as ``out`` (which must not overlap an input).  No function here
synchronises, and each can be captured into a CUDA graph.  Gradients are those of reverse mode;
forward-mode differentiation is refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _cabi
from ._core import _apart, _glue, _launch, device_status_words

_ELEM = {torch.bfloat16: _cabi.OUT_BF16, torch.float16: _cabi.OUT_F16, torch.float32: _cabi.OUT_F32}


class TokenPlan(NamedTuple):
    """Where the pairs (token, slot) of a routing went; int32 CUDA tensors."""
    dest: torch.Tensor       # [T, top_k] row of each pair, -1 for a pair without one
    m_indices: torch.Tensor  # [rows] expert of each row, -1 for rows that stand for no pair
    counts: torch.Tensor     # [E] pairs of each expert
    offsets: torch.Tensor    # [E] first row of each expert
    m_total: torch.Tensor    # [1] end of the last expert's rows, padding included


def sort_capacity(pairs: int, num_experts: int, align: int = 128) -> int:
    """Rows that hold every routing of ``pairs`` pairs: each expert in use ends in a padded block."""
    if pairs < 0 or num_experts < 1 or align < 1:
        raise ValueError(f"bad sizes: pairs={pairs} num_experts={num_experts} align={align}")
    return (pairs + min(num_experts, pairs) * (align - 1)) // align * align


def _rows_arg(t: torch.Tensor, name: str, what: str) -> torch.Tensor:
    """A [rows, H] CUDA tensor of a type the kernels know, its rows whole (they may lie apart)."""
    if not t.is_cuda:
        raise RuntimeError(f"{what}: {name} must be a CUDA tensor (there is no CPU implementation)")
    if t.dim() != 2 or t.dtype not in _ELEM:
        raise ValueError(f"{what}: {name} must be a bf16, fp16 or fp32 [rows, H] tensor, got {t.dtype} {tuple(t.shape)}")
    if t.shape[1] < 1:
        raise ValueError(f"{what}: {name} has no columns")
    if t.stride(1) != 1 and t.shape[1] > 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: the rows of {name} must be contiguous and apart, got strides {tuple(t.stride())}")
    return t


def _grad_arg(t: torch.Tensor) -> torch.Tensor:
    """A gradient as autograd hands it over: expanded and transposed ones are laid out first."""
    return t if t.dim() == 2 and t.stride(1) == 1 and (t.shape[0] < 2 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether one of them carries a tangent of forward-mode differentiation (which the autograd functions
    below refuse: the native path would drop it)."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _int_arg(t: torch.Tensor, shape, device, name: str, what: str) -> torch.Tensor:
    if t.device != device or t.dtype != torch.int32 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} must be int32 {tuple(shape)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _out_arg(out: torch.Tensor, like: torch.Tensor, shape, what: str) -> torch.Tensor:
    if out.device != like.device or out.dtype != like.dtype or tuple(out.shape) != tuple(shape) or not out.is_contiguous():
        raise ValueError(f"{what}: out must be a contiguous {like.dtype} {tuple(shape)} tensor on {like.device}")
    return out


def _sort(x, topk_ids, num_experts, align, out):
    # the native glue does all of this if nothing is unusual; otherwise it has done nothing
    if _glue is not None and (made := _glue.sort_tokens(x, topk_ids, num_experts, align, out)) is not None:
        return made
    what = "sort_tokens"
    _rows_arg(x, "x", what)
    if topk_ids.device != x.device or topk_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: topk_ids must be int32 or int64 on {x.device}, got {topk_ids.dtype} on {topk_ids.device}")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or not 1 <= topk_ids.shape[1] <= _cabi.MAX_TOP_K:
        raise ValueError(f"{what}: topk_ids must be [{x.shape[0]}, 1..{_cabi.MAX_TOP_K}], got {tuple(topk_ids.shape)}")
    if not 1 <= num_experts <= _cabi.MAX_GROUPS or align < 1:
        raise ValueError(f"{what}: num_experts must be 1..{_cabi.MAX_GROUPS} and align positive, got {num_experts} and {align}")
    t, k = (int(v) for v in topk_ids.shape)
    h = int(x.shape[1])
    cap = sort_capacity(t * k, num_experts, align)
    if cap > 0x7fffffff:
        raise ValueError(f"{what}: {cap} rows are more than an int32 row number reaches")
    ids = topk_ids if topk_ids.is_contiguous() else topk_ids.contiguous()
    dev = x.device
    rows = torch.empty((cap, h), dtype=x.dtype, device=dev) if out is None else _out_arg(out, x, (cap, h), what)
    if out is not None:
        _apart(out, what, x=x, topk_ids=ids)
    # tensors of their own (views of one buffer would share a version: writing counts would spoil the saved dest)
    dest, m_indices, counts, offsets, m_total = (torch.empty(size, dtype=torch.int32, device=dev)
                                                 for size in ((t, k), cap, num_experts, num_experts, 1))
    need = int(_cabi.lib.dg_token_sort_scratch_bytes(t, k, num_experts))
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    args = _cabi.TokenSortArgs(
        elem_bytes=x.element_size(), ids64=int(ids.dtype == torch.int64), num_tokens=t, top_k=k, num_groups=int(num_experts),
        hidden=h, align=int(align), cap=cap, x_stride=x.stride(0) if t > 1 else h, x=x.data_ptr(), ids=ids.data_ptr(), rows=rows.data_ptr(),
        dest=dest.data_ptr(), m_indices=m_indices.data_ptr(), counts=counts.data_ptr(), offsets=offsets.data_ptr(),
        m_total=m_total.data_ptr(), scratch=scratch.data_ptr() if need else None, scratch_bytes=need,
        status=device_status_words(dev).data_ptr(), clear=int(out is None))
    _launch(_cabi.lib.dg_token_sort, args, dev, what)
    return rows, dest, m_indices, counts, offsets, m_total


def _unsort(y, dest, weights, out, what):
    t, k = (int(v) for v in dest.shape)
    h = int(y.shape[1])
    if out is None:
        out = torch.empty((t, h), dtype=y.dtype, device=y.device)
    else:
        _apart(_out_arg(out, y, (t, h), what), what, y=y, dest=dest, weights=weights)
    args = _cabi.TokenUnsortArgs(
        elem=_ELEM[y.dtype], num_tokens=t, top_k=k, hidden=h, num_rows=int(y.shape[0]),
        y_stride=y.stride(0) if y.shape[0] > 1 else h, y=y.data_ptr(), dest=dest.data_ptr(),
        weights=weights.data_ptr() if weights is not None else None, out=out.data_ptr())
    _launch(_cabi.lib.dg_token_unsort, args, y.device, what)
    return out


def _plan_args(y, plan, weights, what):
    """The checked (dest, m_indices, weights) of the functions that walk a plan back; y: the sorted rows."""
    _rows_arg(y, "the sorted rows", what)
    return _plan_of(y.shape[0], y.device, plan, weights, what)


def _plan_of(num_rows, device, plan, weights, what):
    if plan.dest.dim() != 2:
        raise ValueError(f"{what}: plan.dest must be [T, top_k], got {tuple(plan.dest.shape)}")
    dest = _int_arg(plan.dest, plan.dest.shape, device, "plan.dest", what)
    m_indices = _int_arg(plan.m_indices, (num_rows,), device, "plan.m_indices", what)
    if weights is not None:
        if weights.device != device or weights.dtype != torch.float32 or weights.shape != plan.dest.shape:
            raise ValueError(f"{what}: weights must be fp32 {tuple(plan.dest.shape)} on {device}, "
                             f"got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
        weights = weights if weights.is_contiguous() else weights.contiguous()
    return dest, m_indices, weights


def sort_tokens_grad(drows: torch.Tensor, plan: TokenPlan) -> torch.Tensor:
    """Gradient of ``sort_tokens`` with respect to its tokens: ``dx[t] = sum_j drows[dest[t, j]]``,
    summed in fp32 and in order.  Rows that stand for no pair are not read."""
    if _glue is not None and (dx := _glue.unsort_tokens(drows, plan.dest, plan.m_indices, None, None)) is not None:
        return dx
    dest, _, _ = _plan_args(drows, plan, None, "sort_tokens_grad")
    return _unsort(drows, dest, None, None, "sort_tokens_grad")


def unsort_tokens_grad(dout: torch.Tensor, y: Optional[torch.Tensor], plan: TokenPlan, weights: Optional[torch.Tensor] = None, *,
                       need_dweights: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of ``unsort_tokens`` (with the whole plan: every row with ``m_indices >= 0`` is named
    by one pair): ``dy[dest[t, j]] = weights[t, j] * dout[t]`` (zero in rows that
    stand for no pair) and ``dweights[t, j] = <dout[t], y[dest[t, j]]>`` in fp32 (zero for a pair
    without a row; None without weights).  Only ``dweights`` reads y: without it y may be None."""
    if _glue is not None and (made := _glue.unsort_tokens_grad(dout, y, plan.dest, plan.m_indices, weights, need_dweights)) is not None:
        return made
    what = "unsort_tokens_grad"
    if y is not None:
        dest, m_indices, weights = _plan_args(y, plan, weights, what)
        _rows_arg(dout, "dout", what)
        if dout.device != y.device or dout.dtype != y.dtype or tuple(dout.shape) != (dest.shape[0], y.shape[1]):
            raise ValueError(f"{what}: dout must be {y.dtype} {(dest.shape[0], y.shape[1])} on {y.device}, "
                             f"got {dout.dtype} {tuple(dout.shape)} on {dout.device}")
    else:
        if weights is not None and need_dweights:
            raise ValueError(f"{what}: the gradient of the weights needs y")
        _rows_arg(dout, "dout", what)
        dest, m_indices, weights = _plan_of(plan.m_indices.numel(), dout.device, plan, weights, what)
        if dout.shape[0] != dest.shape[0]:
            raise ValueError(f"{what}: dout must have {dest.shape[0]} rows, got {tuple(dout.shape)}")
    t, k = (int(v) for v in dest.shape)
    h, rows = int(dout.shape[1]), int(m_indices.shape[0])
    dy = torch.empty((rows, h), dtype=dout.dtype, device=dout.device)
    dw = torch.empty((t, k), dtype=torch.float32, device=dout.device) if weights is not None and need_dweights else None
    args = _cabi.TokenUnsortGradArgs(
        elem=_ELEM[dout.dtype], num_tokens=t, top_k=k, hidden=h, num_rows=rows, clear=1,
        y_stride=y.stride(0) if y is not None and rows > 1 else h, dout_stride=dout.stride(0) if t > 1 else h,
        dout=dout.data_ptr(), y=y.data_ptr() if y is not None else None, dest=dest.data_ptr(),
        weights=weights.data_ptr() if weights is not None else None, m_indices=m_indices.data_ptr(), dy=dy.data_ptr(), dw=dw.data_ptr() if dw is not None else None)
    _launch(_cabi.lib.dg_token_unsort_grad, args, dout.device, what)
    return dy, dw


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, topk_ids, num_experts, align):
        made = _sort(x, topk_ids, num_experts, align, None)
        ctx.mark_non_differentiable(*made[1:])
        ctx.save_for_backward(made[1])
        return made

    @staticmethod
    @once_differentiable
    def backward(ctx, drows, *_):
        dest, = ctx.saved_tensors
        return _unsort(_grad_arg(drows), dest, None, None, "sort_tokens backward"), None, None, None


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, dest, m_indices):
        # only the gradient of the weights reads y, the largest tensor of a layer
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, weights, dest, m_indices)
        return _unsort(y, dest, weights, None, "unsort_tokens")

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, weights, dest, m_indices = ctx.saved_tensors
        plan = TokenPlan(dest, m_indices, None, None, None)
        dy, dw = unsort_tokens_grad(_grad_arg(dout), y, plan, weights, need_dweights=ctx.needs_input_grad[1])
        return dy, dw, None, None


def sort_tokens(x: torch.Tensor, topk_ids: torch.Tensor, num_experts: int, *, align: int = 128,
                out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, TokenPlan]:
    """x bf16 / fp16 / fp32 ``[T, H]`` (rows may lie apart), topk_ids int32 / int64 ``[T, top_k]`` ->
    ``(rows [sort_capacity(T * top_k, num_experts, align), H], plan)``: a copy of token t in row
    ``plan.dest[t, j]`` for each of its experts, every expert's rows together and in token order, each
    expert beginning at a multiple of ``align``.  A negative id is a pair without a row (an expert
    that lives elsewhere); an id >= num_experts is treated the same and reported by
    ``check_device_status``.  Differentiable in x.  ``out``: a buffer for the rows (no gradient)."""
    if torch.is_grad_enabled() and x.requires_grad or _has_tangent(x):
        if out is not None:
            raise ValueError("sort_tokens: out cannot be given where a gradient is recorded")
        made = _SortTokens.apply(x, topk_ids, num_experts, align)
    else:
        made = _sort(x, topk_ids, num_experts, align, out)
    return made[0], TokenPlan(*made[1:])


def unsort_tokens(y: torch.Tensor, plan: TokenPlan, weights: Optional[torch.Tensor] = None, *,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * y[plan.dest[t, j]]`` in y's type, summed in fp32 in the order of
    j; y ``[rows, H]`` in the plan's layout, weights fp32 ``[T, top_k]`` or None for ones.  Pairs
    without a row add nothing.  Differentiable in y and weights; the gradient of y is zero in rows
    that stand for no pair."""
    recorded = torch.is_grad_enabled() and (y.requires_grad or weights is not None and weights.requires_grad) or _has_tangent(y, weights)
    if _glue is not None and not recorded and (made := _glue.unsort_tokens(y, plan.dest, plan.m_indices, weights, out)) is not None:
        return made
    dest, m_indices, w = _plan_args(y, plan, weights, "unsort_tokens")
    if recorded:
        if out is not None:
            raise ValueError("unsort_tokens: out cannot be given where a gradient is recorded")
        return _UnsortTokens.apply(y, w, dest, m_indices)
    return _unsort(y, dest, w, out, "unsort_tokens")


def clear_padding_rows(rows: torch.Tensor, m_indices: torch.Tensor, num_groups: int = 0) -> torch.Tensor:
    """Sets the rows with ``m_indices < 0`` to zero, in place.  ``num_groups``: all rows that a contiguous
    grouped GEMM of as many groups leaves unwritten, i.e. also those of a block of 128 rows whose first
    entry names no group."""
    what = "clear_padding_rows"
    if not 0 <= num_groups <= _cabi.MAX_GROUPS:
        raise ValueError(f"{what}: num_groups must be 0..{_cabi.MAX_GROUPS}, got {num_groups}")
    _rows_arg(rows, "rows", what)
    if not rows.is_contiguous():
        raise ValueError(f"{what}: rows must be contiguous")
    m_indices = _int_arg(m_indices, (rows.shape[0],), rows.device, "m_indices", what)
    args = _cabi.ClearRowsArgs(elem=_ELEM[rows.dtype], num_rows=int(rows.shape[0]), hidden=int(rows.shape[1]),
                               num_groups=int(num_groups), rows=rows.data_ptr(), m_indices=m_indices.data_ptr())
    _launch(_cabi.lib.dg_clear_padding_rows, args, rows.device, what)
    return rows
