"""The MoE layer of ``moe_chain`` in bf16, differentiable: the path a training step takes.

``moe_forward`` / ``expert_mlp_contiguous`` run a layer on quantised operands, forward only.  Here the
tokens, the packed bf16 expert weights and the routing weights all receive gradients:

    tokens sorted by expert -> gate/up grouped GEMM -> SiLU(gate) * up -> down grouped GEMM -> weighted
    sum back in token order

Between the passes a layer keeps, for every routed row, a byte for each of its hidden values and of
its gate and up values (``activation_checkpoint``) and the down GEMM's result in bf16; the activation
itself is computed again from the checkpoint.  CUDA tensors only.  A step can be captured into a
CUDA graph, as long as no eager autograd graph of the same leaves is alive meanwhile.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._cabi import KIND_BF16
from ._core import packed_weight_dims
from .activation_checkpoint import Checkpoint, checkpoint_rows, restore_rows, silu_mul_checkpoint, silu_mul_checkpoint_grad
from .grouped_grad import grouped_bf16_input_grad, grouped_bf16_weight_grad
from .m_group_gemm_nt_contiguous import m_grouped_bf16_gemm_nt_contiguous
from .token_sort import clear_padding_rows, sort_tokens, unsort_tokens


class _ExpertMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, w13, w2, m_indices, kind, recorded):
        m = rows.shape[0]
        h = torch.empty((m, w13.shape[2]), dtype=torch.bfloat16, device=rows.device)
        m_grouped_bf16_gemm_nt_contiguous(rows, w13, h, m_indices)
        act, kept = silu_mul_checkpoint(h, kind=kind, m_indices=m_indices)
        del h
        y = torch.empty((m, w2.shape[2]), dtype=torch.bfloat16, device=rows.device)
        m_grouped_bf16_gemm_nt_contiguous(act, w2, y, m_indices)
        clear_padding_rows(y, m_indices, w2.shape[0])
        entered = checkpoint_rows(rows, kind=kind) if recorded and ctx.needs_input_grad[1] else (None, None)
        ctx.save_for_backward(entered[0], entered[1], kept.q, kept.scale, w13, w2, m_indices)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows_q, rows_scale, q, scale, w13, w2, m_indices = ctx.saved_tensors
        need_rows, need_w13, need_w2 = ctx.needs_input_grad[:3]
        dy = dy.contiguous()
        if dy.data_ptr() % 16:  # a piece of a larger gradient, begun where the products cannot read it
            dy = dy.clone()
        drows = dw13 = dw2 = None
        # rows that stand for no pair are neither written here nor read by what follows (rows of a block
        # that names no expert are carried through the activation as they are, and dropped by the products)
        dact = torch.empty((dy.shape[0], w2.shape[1] * 64), dtype=torch.bfloat16, device=dy.device)
        grouped_bf16_input_grad(dy, w2, m_indices, dact)
        dh, act = silu_mul_checkpoint_grad(Checkpoint(q, scale, torch.bfloat16), dact, m_indices=m_indices, need_act=need_w2)
        del dact
        if need_w2:
            dw2 = grouped_bf16_weight_grad(dy, act, m_indices, w2.shape[0], whole_blocks=True)
        if need_w13:
            dw13 = grouped_bf16_weight_grad(dh, restore_rows(Checkpoint(rows_q, rows_scale, torch.bfloat16)), m_indices, w13.shape[0],
                                            whole_blocks=True)
        if need_rows:
            drows = grouped_bf16_input_grad(dh, w13, m_indices)
        return drows, dw13, dw2, None, None, None


def expert_mlp_bf16(rows: torch.Tensor, m_indices: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, *,
                    checkpoint: str = "fp8") -> torch.Tensor:
    """Both GEMMs of the experts with the activation between them, on rows sorted by expert
    (``sort_tokens`` with ``align`` 128 or 256; the first entry of 128 rows names the expert of them
    all): rows bf16 ``[M, K]``, w13 the packed bf16 ``[E, K/64, 2 I, 64]`` (gate rows, then up rows), w2 the packed ``[E, I/64, K_out, 64]`` -> bf16
    ``[M, K_out]``, zero in rows with ``m_indices < 0`` and in blocks of 128 rows whose first entry names
    no expert.  Differentiable in rows, w13 and w2 (their
    gradients have the packed layout); ``checkpoint`` ("fp8" or "int8") is what the rows and the
    activation's inputs are kept in for the backward pass."""
    what = "expert_mlp_bf16"
    if not (rows.is_cuda and w13.is_cuda and w2.is_cuda):
        raise RuntimeError(f"{what}: all tensors must be CUDA tensors (there is no CPU implementation)")
    e, n13, k = packed_weight_dims(w13, KIND_BF16)
    e2, _, inner = packed_weight_dims(w2, KIND_BF16)
    if rows.dim() != 2 or rows.dtype != torch.bfloat16 or rows.shape[1] != k:
        raise ValueError(f"{what}: rows must be bf16 [M, {k}], got {rows.dtype} {tuple(rows.shape)}")
    if e2 != e or n13 != 2 * inner:
        raise ValueError(f"{what}: w13 {tuple(w13.shape)} and w2 {tuple(w2.shape)} do not belong together")
    if checkpoint not in ("fp8", "int8"):
        raise ValueError(f"{what}: checkpoint must be 'fp8' or 'int8', got {checkpoint!r}")
    return _ExpertMlp.apply(rows, w13, w2, m_indices, checkpoint, torch.is_grad_enabled())


def moe_forward_bf16(hidden: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, w13: torch.Tensor,
                     w2: torch.Tensor, *, checkpoint: str = "fp8") -> torch.Tensor:
    """A whole MoE layer on one GPU, differentiable: hidden bf16 ``[T, K]``, topk_ids ``[T, top_k]``,
    topk_weights fp32 ``[T, top_k]``, packed bf16 expert weights as in ``expert_mlp_bf16`` -> bf16
    ``[T, K_out]``.  Gradients for hidden, topk_weights, w13 and w2."""
    rows, plan = sort_tokens(hidden, topk_ids, int(w13.shape[0]), align=128)
    return unsort_tokens(expert_mlp_bf16(rows, plan.m_indices, w13, w2, checkpoint=checkpoint), plan, topk_weights.to(torch.float32))
