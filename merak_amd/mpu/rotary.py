"""Norms of the query and key heads with the rotary embedding, as one differentiable step between the fused QKV
projection (a ``ColumnParallelLinear``) and attention.

The reference leaves this part of a block to the HF model it wraps; the layers here are what surrounds it.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import ops
from .utils import first_derivative_only


class _QKNormRotary(torch.autograd.Function):
    """Saves its inputs only: the norms are recomputed from the rows that the backward reads anyway."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, cos_table, sin_table, positions, n_q_heads, eps):
        q, k = ops.qk_norm_rope(qkv, cos_table, sin_table, positions, n_q_heads, q_weight, k_weight, eps)
        ctx.save_for_backward(qkv, q_weight, k_weight, cos_table, sin_table, positions)
        ctx.n_q_heads, ctx.eps = n_q_heads, eps
        hd = cos_table.shape[1]
        v = qkv.view(qkv.shape[0], n_q_heads + 2 * k.shape[1], hd)[:, n_q_heads + k.shape[1]:]
        return q, k, v

    @staticmethod
    @first_derivative_only
    def backward(ctx, dq, dk, dv):
        qkv, q_weight, k_weight, cos_table, sin_table, positions = ctx.saved_tensors
        want_dw = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dqkv, dqw, dkw = ops.qk_norm_rope_bwd(dq, dk, dv, qkv, cos_table, sin_table, positions, q_weight, k_weight, ctx.eps,
                                              ctx.n_q_heads, want_dw)
        return dqkv, dqw, dkw, None, None, None, None, None


def qk_norm_rotary(qkv: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                   n_q_heads: int, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                   eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (q [..., n_q, head_dim], k [..., n_kv, head_dim], v): RMSNorm of each query and key head of ``qkv``
    [..., (n_q + 2 n_kv) * head_dim] with ``q_weight`` / ``k_weight`` [head_dim] (None: no norm) and the rotary embedding at
    ``positions`` (int64, the leading dimensions of ``qkv``), with gradients for ``qkv`` and the weights.  ``v`` is a view
    of ``qkv`` (of its contiguous copy, if it was not)."""
    lead, hd = qkv.shape[:-1], cos_table.shape[-1]
    if positions.shape != lead:
        raise ValueError(f"qk_norm_rotary: positions {tuple(positions.shape)} for rows {tuple(lead)}")
    flat = qkv.reshape(-1, qkv.shape[-1])
    q, k, v = _QKNormRotary.apply(flat if flat.is_contiguous() else flat.contiguous(), q_weight, k_weight, cos_table,
                                  sin_table, positions.reshape(-1), n_q_heads, eps)
    n_kv = k.shape[1]
    return q.view(*lead, n_q_heads, hd), k.view(*lead, n_kv, hd), v.view(*lead, n_kv, hd)
