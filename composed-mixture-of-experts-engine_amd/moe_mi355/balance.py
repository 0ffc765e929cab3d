"""Differentiable load balance within sequences (padding left out).

``balance_loss`` is the differentiable form of :func:`moe_mi355.ops.balance_loss_forward`: the mean over the sequences of a
batch of sum_e f_e P_e, with f the shares of the sequence's choices and P its mean probabilities, over valid tokens, and the
z-loss over the valid tokens of the batch.  The router's own aux and z losses (:class:`moe_mi355.router.RouterCore`) are over
every token of the batch, padding included.  The reference has neither (its z-loss is a detached Python float,
moe-engine/pkg/kernels/moe_router.py L:603-612).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops


class BalanceLossFn(torch.autograd.Function):
    """(logits [N,E] f32, idx [N,K], seq_offsets|None, token_mask|None, balance_coef, z_coef) ->
    (balance, z, counts [S,E], tokens [S+2], mean_prob [S,E]); gradients of balance and z reach the logits."""

    @staticmethod
    def forward(ctx, logits, idx, seq_offsets, token_mask, balance_coef: float, z_coef: float):
        balance, z, counts, tokens, mean_prob = ops.balance_loss_forward(logits, idx, seq_offsets, token_mask, balance_coef,
                                                                         z_coef)
        ctx.save_for_backward(logits, counts, tokens, seq_offsets, token_mask)
        ctx.k, ctx.coefs = idx.shape[1], (float(balance_coef), float(z_coef))
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(counts, tokens, mean_prob)
        return balance, z, counts, tokens, mean_prob

    @staticmethod
    def backward(ctx, g_balance, g_z, g_counts, g_tokens, g_mean):
        if (g_balance is None and g_z is None) or not ctx.needs_input_grad[0]:
            return None, None, None, None, None, None
        logits, counts, tokens, seq_offsets, token_mask = ctx.saved_tensors
        # an output that got no gradient contributes no term
        bc = ctx.coefs[0] if g_balance is not None else 0.0
        zc = ctx.coefs[1] if g_z is not None else 0.0
        d = ops.balance_loss_backward(logits, counts, tokens, ctx.k, seq_offsets, token_mask, g_balance, g_z, bc, zc)
        return d, None, None, None, None, None


def balance_loss(logits: torch.Tensor, idx: torch.Tensor, seq_offsets: Optional[torch.Tensor] = None,
                 token_mask: Optional[torch.Tensor] = None, balance_coef: float = 1.0, z_coef: float = 0.0):
    """``(balance, z, counts, tokens, mean_prob)`` as :func:`moe_mi355.ops.balance_loss_forward`, differentiable in the
    logits (those of a router called with ``diff_logits=True``, or any float32 [N, E])."""
    return BalanceLossFn.apply(logits, idx, seq_offsets, token_mask, float(balance_coef), float(z_coef))
