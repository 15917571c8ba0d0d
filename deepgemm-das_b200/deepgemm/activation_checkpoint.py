"""Activation checkpoints in 8 bits, and their use in the backward pass.

A training step keeps, for its backward pass, the inputs of the experts' activation and of the
grouped GEMMs.  In 16 bits they are most of a layer's memory; here they are kept in a byte each with
one fp32 scale for 128 columns, written in the pass that reads the values anyway, and the backward
pass of the activation computes from the checkpoint directly.  ``silu_mul_quant`` is the serving
counterpart: it quantises the activation for the next GEMM and keeps nothing.  CUDA tensors only.

``"fp8"`` (e4m3): the scale is the smallest power of two that brings a block's largest value to 448
or less, and a value comes back within 2^-4 of itself or 2^-10 scales, whichever is more (codes are
subnormal below 2^-6 scales, i.e. 2^-13.8 to 2^-14.8 of the largest); taking rows out again in bf16
adds no rounding.  ``"int8"``: the scale is a 127th of the largest value, and a value comes back within
half of that.  A block that holds a NaN or an infinity comes back as NaN.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _cabi
from ._cabi import KIND_E4M3, KIND_I8
from ._core import _glue, _launch
from .token_sort import _ELEM, _grad_arg, _int_arg, _rows_arg

_CODES = {"fp8": (KIND_E4M3, torch.float8_e4m3fn), "int8": (KIND_I8, torch.int8)}
_KIND_OF = {torch.float8_e4m3fn: KIND_E4M3, torch.int8: KIND_I8}
SCALE_COLUMNS = 128  # columns that share a scale


class Checkpoint(NamedTuple):
    """Rows in 8 bits: ``q[r, c] * scale[r, block of c]`` is what is held; ``dtype`` is what it was."""
    q: torch.Tensor      # [M, H] e4m3 or int8
    scale: torch.Tensor  # fp32 [M, blocks of 128 columns]; of silu_mul_checkpoint: gate's blocks, then up's
    dtype: torch.dtype


def _blocks(h: int) -> int:
    return (h + SCALE_COLUMNS - 1) // SCALE_COLUMNS


def _kind(kind: str, what: str):
    if kind not in _CODES:
        raise ValueError(f"{what}: kind must be 'fp8' or 'int8', got {kind!r}")
    return _CODES[kind]


def _check(c: Checkpoint, halves: int, what: str) -> None:
    if not c.q.is_cuda:
        raise RuntimeError(f"{what}: the checkpoint must be on a CUDA device (there is no CPU implementation)")
    if c.q.dim() != 2 or c.q.dtype not in _KIND_OF or not c.q.is_contiguous() or c.q.shape[1] < halves or c.q.shape[1] % halves:
        raise ValueError(f"{what}: q must be a contiguous e4m3 or int8 [M, {'H' if halves == 1 else '2 H'}] tensor, got {c.q.dtype} {tuple(c.q.shape)}")
    want = (c.q.shape[0], halves * _blocks(c.q.shape[1] // halves))
    if c.scale.device != c.q.device or c.scale.dtype != torch.float32 or tuple(c.scale.shape) != want or not c.scale.is_contiguous():
        raise ValueError(f"{what}: scale must be contiguous fp32 {want} on {c.q.device}, got {c.scale.dtype} {tuple(c.scale.shape)} on {c.scale.device}")
    if c.dtype not in _ELEM:
        raise ValueError(f"{what}: the checkpoint's dtype must be bf16, fp16 or fp32, got {c.dtype}")


def checkpoint_rows(x: torch.Tensor, *, kind: str = "fp8") -> Checkpoint:
    """x bf16 / fp16 / fp32 ``[M, H]`` (rows may lie apart) -> its checkpoint."""
    what = "checkpoint_rows"
    code, qdtype = _kind(kind, what)
    if _glue is not None and (made := _glue.checkpoint_rows(x, code)) is not None:
        return Checkpoint(*made, x.dtype)
    _rows_arg(x, "x", what)
    m, h = (int(v) for v in x.shape)
    q = torch.empty((m, h), dtype=qdtype, device=x.device)
    scale = torch.empty((m, _blocks(h)), dtype=torch.float32, device=x.device)
    args = _cabi.CheckpointArgs(elem=_ELEM[x.dtype], kind=code, num_rows=m, hidden=h, x_stride=x.stride(0) if m > 1 else h,
                                x=x.data_ptr(), q=q.data_ptr(), scale=scale.data_ptr())
    _launch(_cabi.lib.dg_checkpoint_rows, args, x.device, what)
    return Checkpoint(q, scale, x.dtype)


def restore_rows(checkpoint: Checkpoint) -> torch.Tensor:
    """The rows that a checkpoint holds, in the type they had: ``q * scale``, rounded once and at most
    the type's largest finite value."""
    what = "restore_rows"
    if _glue is not None and checkpoint.dtype in _ELEM and \
            (made := _glue.restore_rows(checkpoint.q, checkpoint.scale, _ELEM[checkpoint.dtype])) is not None:
        return made
    _check(checkpoint, 1, what)
    q, scale, dtype = checkpoint
    m, h = (int(v) for v in q.shape)
    x = torch.empty((m, h), dtype=dtype, device=q.device)
    args = _cabi.CheckpointArgs(elem=_ELEM[dtype], kind=_KIND_OF[q.dtype], num_rows=m, hidden=h, x_stride=h, x=x.data_ptr(),
                                q=q.data_ptr(), scale=scale.data_ptr())
    _launch(_cabi.lib.dg_restore_rows, args, q.device, what)
    return x


def silu_mul_checkpoint(x: torch.Tensor, *, kind: str = "fp8", m_indices: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, Checkpoint]:
    """x ``[M, 2 H]``, gate in the first H columns, up in the others -> ``(act [M, H], checkpoint of x)``:
    ``act = gate * sigmoid(gate) * up`` in fp32 from x itself, rounded once (16-bit types: a sigmoid below
    2^-126, i.e. of a gate below -87.3, counts as zero).  Rows with ``m_indices < 0``
    are not read; their ``act`` is zero and their checkpoint holds zeros."""
    what = "silu_mul_checkpoint"
    code, qdtype = _kind(kind, what)
    if _glue is not None and (made := _glue.silu_mul_checkpoint(x, code, m_indices)) is not None:
        return made[0], Checkpoint(made[1], made[2], x.dtype)
    _rows_arg(x, "x", what)
    if x.shape[1] % 2:
        raise ValueError(f"{what}: the rows of x must hold a gate and an up half, got {x.shape[1]} columns")
    m, h = int(x.shape[0]), int(x.shape[1]) // 2
    if m_indices is not None:
        m_indices = _int_arg(m_indices, (m,), x.device, "m_indices", what)
    act = torch.empty((m, h), dtype=x.dtype, device=x.device)
    q = torch.empty((m, 2 * h), dtype=qdtype, device=x.device)
    scale = torch.empty((m, 2 * _blocks(h)), dtype=torch.float32, device=x.device)
    args = _cabi.ActCheckpointArgs(elem=_ELEM[x.dtype], kind=code, num_rows=m, hidden=h, clear=1,
                                   x_stride=x.stride(0) if m > 1 else 2 * h, x=x.data_ptr(), q=q.data_ptr(),
                                   scale=scale.data_ptr(), act=act.data_ptr(),
                                   m_indices=m_indices.data_ptr() if m_indices is not None else None)
    _launch(_cabi.lib.dg_act_checkpoint, args, x.device, what)
    return act, Checkpoint(q, scale, x.dtype)


def silu_mul_checkpoint_grad(checkpoint: Checkpoint, dact: torch.Tensor, *, m_indices: Optional[torch.Tensor] = None,
                             need_act: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(dx [M, 2 H], act [M, H])`` from the checkpoint of ``silu_mul_checkpoint`` and the gradient of its
    result: the gradients of gate and up at the values the checkpoint holds, and the activation of
    those values once more (what the weight gradient behind it multiplies; None unless asked for).
    Rows with ``m_indices < 0`` are zero in both, whatever ``dact`` holds there."""
    what = "silu_mul_checkpoint_grad"
    if _glue is not None and dact.dtype == checkpoint.dtype and \
            (made := _glue.silu_mul_checkpoint_grad(checkpoint.q, checkpoint.scale, dact, m_indices, need_act)) is not None:
        return made
    _check(checkpoint, 2, what)
    q, scale, dtype = checkpoint
    m, h = int(q.shape[0]), int(q.shape[1]) // 2
    _rows_arg(dact, "dact", what)
    if dact.device != q.device or dact.dtype != dtype or tuple(dact.shape) != (m, h):
        raise ValueError(f"{what}: dact must be {dtype} {(m, h)} on {q.device}, got {dact.dtype} {tuple(dact.shape)} on {dact.device}")
    if m_indices is not None:
        m_indices = _int_arg(m_indices, (m,), q.device, "m_indices", what)
    dx = torch.empty((m, 2 * h), dtype=dtype, device=q.device)
    act = torch.empty((m, h), dtype=dtype, device=q.device) if need_act else None
    args = _cabi.ActCheckpointArgs(elem=_ELEM[dtype], kind=_KIND_OF[q.dtype], num_rows=m, hidden=h, clear=1,
                                   dact_stride=dact.stride(0) if m > 1 else h, dact=dact.data_ptr(), q=q.data_ptr(),
                                   scale=scale.data_ptr(), act=act.data_ptr() if act is not None else None, dx=dx.data_ptr(),
                                   m_indices=m_indices.data_ptr() if m_indices is not None else None)
    _launch(_cabi.lib.dg_act_checkpoint_grad, args, q.device, what)
    return dx, act


class _SiluMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, m_indices):
        act, kept = silu_mul_checkpoint(x, kind=kind, m_indices=m_indices)
        ctx.save_for_backward(kept.q, kept.scale, m_indices)
        ctx.dtype = x.dtype
        return act

    @staticmethod
    @once_differentiable
    def backward(ctx, dact):
        q, scale, m_indices = ctx.saved_tensors
        dx, _ = silu_mul_checkpoint_grad(Checkpoint(q, scale, ctx.dtype), _grad_arg(dact), m_indices=m_indices, need_act=False)
        return dx, None, None


def silu_mul(x: torch.Tensor, *, checkpoint: str = "fp8", m_indices: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``silu_mul_checkpoint`` with its gradient: differentiable in x, keeping a byte for each of its
    values instead of x."""
    return _SiluMul.apply(x, checkpoint, m_indices)
