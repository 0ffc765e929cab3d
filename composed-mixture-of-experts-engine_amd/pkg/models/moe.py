"""``RMSNorm`` and ``ToyMoEBlock`` (moe-engine/pkg/models/moe.py L:63-126) on the fused kernels.

``ToyMoEBlock.forward`` is ``x + moe(norm(x))`` (L:125-126).  Here the norm and the router run as one
operation (:class:`moe_mi355.norm.NormRouterCore`): the hidden state is read once for both, the router
routes the bf16-rounded normalised rows exactly as it would route ``norm(x)``, and the expert path takes
those same rows.  Modules whose experts are not the built-in SwiGLU, or shapes the norm kernels do not
take, use the plain composition ``moe(norm(x))``.

In a stack the sum ``x + moe(norm(x))`` is read again by the next block's norm.  With ``residual`` the sum is left to that norm:
``out, h = block(x, residual=r)`` is ``h = x + r``, ``out = moe(norm(h))``, the addition inside the norm's kernel; the next block
takes ``(out, residual=h)`` and the last norm (``RMSNorm.forward(out, residual=h)``) adds the last one.  ``forward_int8`` and
``forward_fp8`` serve a block on experts in 8 bits, whose rows the norm writes quantized.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from moe_mi355 import ops
from moe_mi355.norm import RMSNormFn, RMSNormResidualFn
from pkg.distributed.moe_layer import DistributedMoELayer

_NORM_MAX_H = 8192


class RMSNorm(nn.Module):
    """Root-mean-square layer normalisation (L:63-86): ``weight`` [dim] (ones), ``eps`` (1e-5).

    ``forward(x)`` returns ``((x * rsqrt(mean(x^2, -1) + eps)) * weight).to(x.dtype)`` with fp32 arithmetic,
    one HIP kernel (the reference's torch composition makes several fp32 passes)."""

    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def extra_repr(self) -> str:
        return f"dim={self.weight.shape[0]}, eps={self.eps}"

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """The normalised ``x``; with ``residual`` (of x's shape and dtype) ``(norm(h), h)`` for ``h = x + residual``."""
        H = x.shape[-1]
        if residual is None:
            return RMSNormFn.apply(x.reshape(-1, H), self.weight, self.eps).reshape(x.shape)
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
        return RMSNormResidualFn.apply(x, residual, self.weight, self.eps)

    @torch.no_grad()
    def quantized(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, fmt: str = "int8"):
        """For serving: ``(q, scale, norm(h), h)`` with the normalised rows in 8 bits too (:func:`moe_mi355.ops.rmsnorm_quant`;
        ``q`` [N, H], ``scale`` [N] over the flattened rows, the others in x's shape); h is x without ``residual``."""
        H = x.shape[-1]
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
        q, scale, xn, h = ops.rmsnorm_quant(x.reshape(-1, H), self.weight, self.eps,
                                            None if residual is None else residual.reshape(-1, H), fmt=fmt, keep_norm=True)
        return q, scale, xn.reshape(x.shape), (x if h is None else h.reshape(x.shape))


class ToyMoEBlock(nn.Module):
    """Single MoE transformer block: RMSNorm + DistributedMoELayer + residual (L:89-126)."""

    def __init__(
        self,
        hidden_dim: int,
        ffn_dim: int,
        num_experts: int,
        top_k: int,
        topology,
        capacity_factor: float = 1.25,
        dtype: torch.dtype = torch.float32,
        **layer_kwargs,
    ):
        super().__init__()
        self.norm = RMSNorm(hidden_dim)
        self.moe = DistributedMoELayer(
            hidden_dim=hidden_dim,
            ffn_dim=ffn_dim,
            num_experts=num_experts,
            top_k=top_k,
            topology=topology,
            capacity_factor=capacity_factor,
            dtype=dtype,
            **layer_kwargs,
        )

    def _fused(self, x: torch.Tensor) -> bool:
        return (
            x.is_cuda
            and x.shape[-1] <= _NORM_MAX_H
            and x.shape[-1] % 8 == 0
            and x.dtype in (torch.float32, torch.bfloat16)
            and self.norm.weight.dtype in (torch.float32, torch.bfloat16)
            and self.moe.router.gate_w.dtype == x.dtype
        )

    def forward(self, x: torch.Tensor, seq_offsets=None, token_mask=None, residual: Optional[torch.Tensor] = None):
        """``seq_offsets`` and ``token_mask``: the sequences and valid tokens of the router's balance loss
        (:meth:`DistributedMoELayer.forward`).  With ``residual``, ``(moe(norm(h)), h)`` for ``h = x + residual``."""
        if residual is not None:
            xn, h = self.norm(x, residual)
            return self.moe(xn, seq_offsets, token_mask), h
        if self._fused(x):
            out = self.moe.forward_normed(x, self.norm.weight, self.norm.eps, seq_offsets, token_mask)
        else:
            out = self.moe(self.norm(x), seq_offsets, token_mask)
        return x + out

    @torch.no_grad()
    def forward_int8(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, seq_offsets=None, token_mask=None):
        """``forward`` for serving on the layer's int8 weights (:meth:`DistributedMoELayer.forward_int8`), the experts' rows
        quantized by the norm from its fp32 values: ``x + moe(norm(x))``, or with ``residual`` ``(moe(norm(h)), h)``."""
        return self._serve(self.moe._forward_int8, "int8", x, residual, seq_offsets, token_mask)

    @torch.no_grad()
    def forward_fp8(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, seq_offsets=None, token_mask=None):
        """The same on e4m3 rows and weights (:meth:`DistributedMoELayer.forward_fp8`)."""
        return self._serve(self.moe._forward_fp8, "e4m3", x, residual, seq_offsets, token_mask)

    def _serve(self, layer, fmt, x, residual, seq_offsets, token_mask):
        if x.dim() not in (2, 3):
            raise ValueError(f"tokens must be rank 2 or 3, got {x.dim()}")
        q, scale, xn, h = self.norm.quantized(x, residual, fmt)
        out = layer(xn.reshape(-1, x.shape[-1]), x.shape, seq_offsets, token_mask, quantized=(q, scale)).reshape(x.shape)
        return x + out if residual is None else (out, h)
