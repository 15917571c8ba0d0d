"""Gradients of the contiguous BF16 grouped GEMM ``y[i] = x[i] @ W[m_indices[i]]^T``
(``m_grouped_bf16_gemm_nt_contiguous``), on the packed weight the forward pass uses:

* ``grouped_bf16_input_grad``:  ``dx[i] = dy[i] @ W[m_indices[i]]``
* ``grouped_bf16_weight_grad``: ``dW[g] = sum of dy[i]^T x[i]`` over the rows of group g, in the packed
  layout ``[G, K/64, N, 64]`` of the weight, so that an optimiser steps over both element by element
  (``unpack_weight`` gives the plain ``[G, N, K]`` form).

Both read one group for every 128 rows from ``m_indices``, named by the first of them, as the forward
product does; rows with ``m_indices < 0`` stand for nothing, whatever they hold.  They are the
product's gradients for blocks whose other entries are that group's or negative, as ``sort_tokens``
lays them out.  Where an entry names another group, the forward product and the input gradient take
the row with the block's group all the same; the weight gradient leaves it out, unless it is asked to
take ``whole_blocks``.  An ``out`` must not overlap an input.  CUDA tensors only.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _cabi
from ._cabi import KIND_BF16
from ._core import _apart, _glue, _launch, device_status_words, packed_weight_dims


def _bf16_rows(t: torch.Tensor, name: str, what: str) -> torch.Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"{what}: {name} must be a CUDA tensor (there is no CPU implementation)")
    if t.dim() != 2 or t.dtype != torch.bfloat16 or not t.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be a contiguous bf16 [M, columns] tensor, got {t.dtype} {tuple(t.shape)}")
    if t.data_ptr() % 16:
        raise RuntimeError(f"{what}: {name} must start on a 16-byte boundary")
    return t


def _indices(m_indices: torch.Tensor, rows: torch.Tensor, what: str) -> None:
    if m_indices.device != rows.device or m_indices.dtype != torch.int32 or not m_indices.is_contiguous() \
            or m_indices.dim() != 1 or m_indices.numel() != rows.shape[0]:
        raise RuntimeError(f"{what}: m_indices must be contiguous int32 [{rows.shape[0]}] on {rows.device}")


def grouped_bf16_input_grad(dy: torch.Tensor, weight: torch.Tensor, m_indices: torch.Tensor,
                            out: Optional[torch.Tensor] = None, *, block_n: int = 0) -> torch.Tensor:
    """dy bf16 ``[M, N]``, weight the packed bf16 ``[G, K/64, N, 64]`` -> dx bf16 ``[M, K]``.  Rows with
    ``m_indices < 0``, and those of a block whose first entry names no group, are zero, or, in a given
    ``out``, left as they are."""
    what = "grouped_bf16_input_grad"
    if _glue is not None and (made := _glue.input_grad(dy, weight, m_indices, out, block_n)) is not None:
        return made
    _bf16_rows(dy, "dy", what)
    g, n, k = packed_weight_dims(weight, KIND_BF16)
    if weight.device != dy.device or weight.dtype != torch.bfloat16 or not weight.is_contiguous():
        raise RuntimeError(f"{what}: weight must be a contiguous bf16 tensor on {dy.device}")
    if weight.data_ptr() % 16:
        raise RuntimeError(f"{what}: weight must start on a 16-byte boundary")
    m = int(dy.shape[0])
    if dy.shape[1] != n:
        raise RuntimeError(f"{what}: dy has {dy.shape[1]} columns, the weight {n} rows")
    _indices(m_indices, dy, what)
    if out is not None:
        _bf16_rows(out, "out", what)
        if out.device != dy.device or tuple(out.shape) != (m, k):
            raise RuntimeError(f"{what}: out must be {(m, k)} on {dy.device}, got {tuple(out.shape)} on {out.device}")
        _apart(out, what, dy=dy, weight=weight, m_indices=m_indices)
    dx = torch.empty((m, k), dtype=torch.bfloat16, device=dy.device) if out is None else out
    args = _cabi.InputGradArgs(dy=dy.data_ptr(), w_packed=weight.data_ptr(), dx=dx.data_ptr(), m_indices=m_indices.data_ptr(),
                               num_groups=g, m_total=m, n=n, k=k, block_n=int(block_n), clear=int(out is None),
                               status=device_status_words(dy.device).data_ptr())
    _launch(_cabi.lib.dg_grouped_input_grad, args, dy.device, what)
    return dx


def grouped_bf16_weight_grad(dy: torch.Tensor, x: torch.Tensor, m_indices: torch.Tensor, num_groups: int, *,
                             out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
                             accumulate: bool = False, tile: int = 0, whole_blocks: bool = False) -> torch.Tensor:
    """dy bf16 ``[M, N]``, x bf16 ``[M, K]`` -> dW ``[G, K/64, N, 64]`` in bf16 or fp32 (``dtype``, or the
    type of ``out``), summed in fp32 over the rows whose entry is the group of their block.
    ``accumulate`` adds to a given fp32 ``out``, for micro-batches; otherwise groups without rows give
    zeros.  ``whole_blocks``: rows with any entry >= 0 count for the group of their block, as in the
    forward product."""
    what = "grouped_bf16_weight_grad"
    if _glue is not None and dtype in (torch.bfloat16, torch.float32) and \
            (made := _glue.weight_grad(dy, x, m_indices, num_groups, out, dtype == torch.float32, accumulate, tile,
                                      whole_blocks)) is not None:
        return made
    _bf16_rows(dy, "dy", what)
    _bf16_rows(x, "x", what)
    if x.device != dy.device or x.shape[0] != dy.shape[0]:
        raise RuntimeError(f"{what}: x must have the rows of dy on its device, got {tuple(x.shape)} on {x.device}")
    _indices(m_indices, dy, what)
    m, n, k = int(dy.shape[0]), int(dy.shape[1]), int(x.shape[1])
    if n < 16 or n % 16 or k < 64 or k % 64:
        raise RuntimeError(f"{what}: dy needs a multiple of 16 columns and x one of 64, got {n} and {k}")
    if out is None:
        if accumulate:
            raise ValueError(f"{what}: accumulate needs an out to add to")
        out = torch.empty((num_groups, k // 64, n, 64), dtype=dtype, device=dy.device)
    if out.device != dy.device or tuple(out.shape) != (num_groups, k // 64, n, 64) or not out.is_contiguous() \
            or out.dtype not in (torch.bfloat16, torch.float32) or out.data_ptr() % 16:
        raise RuntimeError(f"{what}: the gradient must be a contiguous bf16 or fp32 {(num_groups, k // 64, n, 64)} tensor on "
                           f"{dy.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
    if accumulate and out.dtype != torch.float32:
        raise ValueError(f"{what}: a gradient is added to in fp32, got {out.dtype}")
    _apart(out, what, dy=dy, x=x, m_indices=m_indices)
    args = _cabi.WeightGradArgs(dy=dy.data_ptr(), x=x.data_ptr(), dw=out.data_ptr(), m_indices=m_indices.data_ptr(),
                                num_groups=int(num_groups), m_total=m, n=n, k=k,
                                out_kind=_cabi.OUT_F32 if out.dtype == torch.float32 else _cabi.OUT_BF16,
                                accumulate=int(accumulate), tile=int(tile), whole_blocks=int(whole_blocks),
                                status=device_status_words(dy.device).data_ptr())
    _launch(_cabi.lib.dg_grouped_weight_grad, args, dy.device, what)
    return out
