"""MoE layer with the reference's API, on the gfx950 kernels.

Mirrors ``moe-engine/pkg/distributed/moe_layer.py``:

* ``DistributedMoELayer(hidden_dim, ffn_dim, num_experts, top_k, topology,
  capacity_factor=1.25, capacity_dropping=False, dtype=torch.float32)``,
  ``forward([B,S,H] | [N,H]) -> same shape`` (L:206-360);
* ``compute_capacity_drop_mask(idx, num_experts, capacity) -> Bool[N,K]``
  and ``_cumcount(groups) -> Long[n]`` (L:64-155);
* ``_SwiGLUExpert`` (L:166-198) and the attributes ``router``, ``experts``,
  ``local_expert_ids``, ``last_{dispatch,combine,expert_compute}_ms``,
  ``last_overlap_ratio``, ``last_dropped_token_fraction``, ``_expert_to_rank``.

Forward pipeline, all on the GPU with no host synchronisation:
router kernel -> planner kernels (capacity drops, row layout) -> permute ->
SwiGLU grouped GEMM -> weighted combine.  The backward is the fused mirror
(combine-bwd, grouped GEMM backward, permute-bwd) plus the router backward.

Row layout (``layout`` argument, new):
* ``"reference"`` (default) reproduces the reference exactly: tokens are
  stable-sorted by their first choice, repeated K times, and the [N*K, H]
  buffer is cut into E equal chunks, chunk i going to expert i whatever the
  router chose (L:317-337); rows past E*chunk contribute zero.
* ``"routed"``: slot (t, k) goes to expert idx[t, k]; dropped slots get no row.

Expert weights are held stacked -- ``w_gate`` / ``w_up`` [E, F, H] and
``w_down`` [E, H, F] -- so one grouped GEMM reads them; ``experts[i]`` exposes
expert i's slices as ``w_gate.weight`` etc., and ``state_dict`` /
``load_state_dict`` use the reference's per-expert keys
(``experts.{i}.w_gate.weight``).  Assigning a different ModuleList to
``experts`` (the reference's extension point) switches the layer to calling
those modules per expert between the dispatch and combine kernels.  bf16 and
fp32 (the reference's default dtype) use the fused HIP grouped GEMM (bf16 or
fp32 MFMA); other dtypes and shapes call the expert modules per expert.
"""

from __future__ import annotations

import contextlib
import math
from typing import List, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from moe_mi355 import ops
from moe_mi355.layer import CombineFn, ExpertsFn, ExpertsMxfp4Fn, PermuteFn
from pkg.kernels.moe_router import MoERouter

__all__ = ["DistributedMoELayer", "compute_capacity_drop_mask", "_cumcount"]

_LAYOUTS = {"reference": ops.LAYOUT_REFERENCE, "routed": ops.LAYOUT_ROUTED}


class _ExpertTimer:
    """Two timing events on the current stream around the expert compute; the elapsed time is read only when
    asked for.  None on the CPU and under graph capture."""

    __slots__ = ("a", "b")

    @classmethod
    def new(cls, like: torch.Tensor) -> Optional["_ExpertTimer"]:
        if not like.is_cuda or torch.cuda.is_current_stream_capturing():
            return None
        t = cls()
        t.a = torch.cuda.Event(enable_timing=True)
        t.b = torch.cuda.Event(enable_timing=True)
        return t

    def start(self) -> None:
        self.a.record()

    def stop(self) -> None:
        self.b.record()

    def elapsed_ms(self) -> float:
        self.b.synchronize()
        return max(float(self.a.elapsed_time(self.b)), 0.0)


# The planner's key tables hold one contiguous range of at most this many ids (and K * E <= 8192 keys).
_PLAN_MAX_KEYS = 1024


def _cumcount(groups: torch.Tensor) -> torch.Tensor:
    """Each element's 0-based position among earlier elements of its group (L:64-115), for any integer ids.

    Ids spanning at most 1024 values run the planner's stable-grouping kernel (one column of K=1); wider
    ranges run moe_cumcount (a stable radix sort of the ids).  One host read of the id range."""
    n = groups.shape[0]
    if n == 0:
        return torch.empty(0, dtype=torch.long, device=groups.device)
    g = groups.reshape(n, 1).long()
    lo, hi = (int(v) for v in torch.stack([g.min(), g.max()]).tolist())
    if hi - lo + 1 > _PLAN_MAX_KEYS:
        return ops.cumcount(g.reshape(-1))
    g = g - lo
    E = hi - lo + 1
    # rank of each element within its key = position in the stable sort minus the key's offset
    p = ops.plan(g, max(E, 1), capacity=-1, layout=ops.LAYOUT_ROUTED)
    pos = p.slot_row.long()
    return pos - p.offsets.long()[g.reshape(-1)]


def compute_capacity_drop_mask(idx: torch.Tensor, num_experts: int, capacity: int) -> torch.Tensor:
    """``drop[t, k] = cumcount(idx[:, k])[t] >= capacity`` per column (L:118-155), for any integer ids."""
    N, K = idx.shape
    if N == 0:
        return torch.zeros(N, K, dtype=torch.bool, device=idx.device)
    if capacity < 0:  # every slot is at a position >= capacity
        return torch.ones(N, K, dtype=torch.bool, device=idx.device)
    # any integer group ids are valid here, as in the reference (one host read of the range)
    lo, hi = (int(v) for v in torch.stack([idx.min(), idx.max()]).tolist())
    if lo < 0 or hi >= num_experts:
        idx = idx - lo
        num_experts = hi - lo + 1
    if num_experts > _PLAN_MAX_KEYS or K * num_experts > 8192 or K > num_experts:
        # ids too many for the planner's key tables: the column ranks from the general kernel
        return torch.stack([_cumcount(idx[:, k]) >= capacity for k in range(K)], dim=1)
    p = ops.plan(idx, num_experts, capacity=int(capacity), layout=ops.LAYOUT_REFERENCE)
    return p.drop


_MXFP4 = ("mxfp4_gate", "mxfp4_up", "mxfp4_down", "mxfp4_gate_scale", "mxfp4_up_scale", "mxfp4_down_scale")
_INT8 = ("int8_gate", "int8_up", "int8_down", "int8_gate_scale", "int8_up_scale", "int8_down_scale")


class _ExpertWeight(nn.Module):
    """``.weight`` of one expert projection: a view of the layer's stacked tensor."""

    def __init__(self, owner_ref, name: str, index: int):
        super().__init__()
        object.__setattr__(self, "_owner", owner_ref)
        object.__setattr__(self, "_name", name)
        object.__setattr__(self, "_index", index)

    @property
    def weight(self) -> torch.Tensor:
        stacked = getattr(self._owner(), self._name)
        if stacked is None:
            raise RuntimeError(f"the layer's {self._name} was dropped: only forward_mxfp4 runs")
        return stacked[self._index]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return F.linear(x, self.weight)


class _SwiGLUExpert(nn.Module):
    """``w_down(silu(w_gate(x)) * w_up(x))`` (L:166-198) over expert ``index``'s slices."""

    def __init__(self, owner_ref, index: int):
        super().__init__()
        self.w_gate = _ExpertWeight(owner_ref, "w_gate", index)
        self.w_up = _ExpertWeight(owner_ref, "w_up", index)
        self.w_down = _ExpertWeight(owner_ref, "w_down", index)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.w_down(F.silu(self.w_gate(x)) * self.w_up(x))


class DistributedMoELayer(nn.Module):
    def __init__(
        self,
        hidden_dim: int,
        ffn_dim: int,
        num_experts: int,
        top_k: int,
        topology,
        capacity_factor: float = 1.25,
        capacity_dropping: bool = False,
        dtype: torch.dtype = torch.float32,
        layout: str = "reference",
        aux_loss_coef: float = 0.0,
        z_loss_coef: float = 0.0,
        check_numerics: bool = True,
        seq_balance_coef: float = 0.0,
    ):
        super().__init__()
        if getattr(topology, "ep_size", 1) != 1 or getattr(topology, "tp_size", 1) != 1:
            raise NotImplementedError("this build runs one GPU's experts; ep_size/tp_size > 1 are out of scope")
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
        self.hidden_dim = hidden_dim
        self.ffn_dim = ffn_dim
        self.num_experts = num_experts
        self.top_k = top_k
        self.topology = topology
        self.capacity_factor = capacity_factor
        self.capacity_dropping = capacity_dropping
        self.layout = layout
        self.check_numerics = check_numerics
        self.local_expert_ids: List[int] = topology.experts_on_this_rank(num_experts)
        dev = getattr(topology, "device", None)
        E = len(self.local_expert_ids)
        # nn.Linear-style init N(0, 1/sqrt(in)) per projection (tensor_parallel.py L:109, L:187)
        self.w_gate = nn.Parameter(torch.empty(E, ffn_dim, hidden_dim, device=dev, dtype=dtype))
        self.w_up = nn.Parameter(torch.empty(E, ffn_dim, hidden_dim, device=dev, dtype=dtype))
        self.w_down = nn.Parameter(torch.empty(E, hidden_dim, ffn_dim, device=dev, dtype=dtype))
        # the experts in 4 bits (quantize_mxfp4, load_mxfp4): they move with the layer and are not in its state_dict, whose
        # keys are the reference's
        for name in _MXFP4:
            self.register_buffer(name, None, persistent=False)
        # and in int8 (quantize_int8, load_int8), the fp32 scales as int32 words: a change of the layer's dtype leaves them alone
        for name in _INT8:
            self.register_buffer(name, None, persistent=False)
        nn.init.normal_(self.w_gate, mean=0.0, std=1.0 / math.sqrt(hidden_dim))
        nn.init.normal_(self.w_up, mean=0.0, std=1.0 / math.sqrt(hidden_dim))
        nn.init.normal_(self.w_down, mean=0.0, std=1.0 / math.sqrt(ffn_dim))
        import weakref

        ref = weakref.ref(self)
        self.experts = nn.ModuleList([_SwiGLUExpert(ref, i) for i in range(E)])
        self.router = MoERouter(hidden_dim, num_experts, top_k, dtype=dtype, aux_loss_coef=aux_loss_coef,
                                z_loss_coef=z_loss_coef, sync_profile=check_numerics,
                                seq_balance_coef=seq_balance_coef)
        if dev is not None:
            self.router.to(dev)
        self.last_dispatch_ms: float = 0.0
        self.last_combine_ms: float = 0.0
        self._expert_ms: float = 0.0
        self._expert_timer: Optional[_ExpertTimer] = None
        self.last_overlap_ratio: float = 0.0
        self.last_plan: Optional[ops.Plan] = None
        self._register_state_dict_hook(DistributedMoELayer._to_reference_keys)
        self._register_load_state_dict_pre_hook(DistributedMoELayer._from_reference_keys, with_module=True)

    # ---- state_dict in the reference's per-expert key format ----
    @staticmethod
    def _to_reference_keys(module, state_dict, prefix, local_metadata):
        for name in ("w_gate", "w_up", "w_down"):
            key = prefix + name
            if key in state_dict:
                stacked = state_dict.pop(key)
                for i in range(stacked.shape[0]):
                    state_dict[f"{prefix}experts.{i}.{name}.weight"] = stacked[i]
        return state_dict

    @staticmethod
    def _from_reference_keys(module, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                             error_msgs):
        for name in ("w_gate", "w_up", "w_down"):
            if getattr(module, name) is None:  # dropped for serving from 4-bit weights
                continue
            keys = [f"{prefix}experts.{i}.{name}.weight" for i in range(getattr(module, name).shape[0])]
            if all(k in state_dict for k in keys):
                state_dict[prefix + name] = torch.stack([state_dict.pop(k) for k in keys])

    @property
    def last_expert_compute_ms(self) -> float:
        """Time of the last forward's expert FFN compute (the grouped GEMMs, or the per-expert module calls),
        measured with device events on the launch stream (moe_layer.py L:326-337 times the same span with the
        host clock).  Reading it waits for the GPU to finish that span."""
        t = self._expert_timer
        if t is not None:
            self._expert_timer = None
            self._expert_ms = t.elapsed_ms()
        return self._expert_ms

    @last_expert_compute_ms.setter
    def last_expert_compute_ms(self, v: float) -> None:
        self._expert_timer = None
        self._expert_ms = float(v)

    @property
    def last_dropped_token_fraction(self) -> float:
        """Fraction of (token, k) slots dropped by capacity in the last forward (reads the device count)."""
        p = self.last_plan
        if p is None or not self.capacity_dropping or p.rows == 0:
            return 0.0
        return float(p.ndrop.item()) / float(p.rows)

    def extra_repr(self) -> str:
        return (
            f"hidden={self.hidden_dim}, num_experts={self.num_experts}, top_k={self.top_k}, "
            f"local_experts={len(self.local_expert_ids)}, ep_size=1, layout={self.layout}"
        )

    def _fused(self) -> bool:
        return (
            # the grouped GEMM's shapes: bf16 H % 8 == 0, fp32 H % 4 == 0, both F % 32 == 0
            self.w_gate is not None
            and self.w_gate.dtype in (torch.bfloat16, torch.float32)
            and self.w_gate.shape[-1] % (8 if self.w_gate.dtype == torch.bfloat16 else 4) == 0
            and self.w_gate.shape[1] % 32 == 0
            and all(type(m) is _SwiGLUExpert and m.w_gate._owner() is self for m in self.experts)
            and len(self.experts) == self.num_experts
        )

    def _router_args(self, flat: torch.Tensor, shape, seq_offsets, token_mask):
        """The router's tokens and its arguments for the balance loss of sequences (the tokens then as [B, S, H]: by default
        the rows are the sequences)."""
        if seq_offsets is None and token_mask is None and getattr(self.router, "seq_balance_coef", 0.0) == 0.0:
            return flat, {}
        return (flat.view(shape) if len(shape) == 3 else flat), {"seq_offsets": seq_offsets, "token_mask": token_mask}

    def forward(self, tokens: torch.Tensor, seq_offsets: Optional[torch.Tensor] = None,
                token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``seq_offsets`` and ``token_mask`` go to the router's balance loss of sequences (:meth:`MoERouter.forward`; the
        rows of a [B, S, H] batch are its sequences unless told otherwise): every token is routed and dispatched."""
        original_shape = tokens.shape
        if tokens.dim() not in (2, 3):
            raise ValueError(f"tokens must be rank 2 or 3, got {tokens.dim()}")
        H = tokens.shape[-1]
        flat = tokens.reshape(-1, H)
        routed, seq = self._router_args(flat, tokens.shape, seq_offsets, token_mask)
        with self._deferred_router_check(), self._linked_tokens():
            idx, weights, _cnt = self.router(routed, **seq)
        # the router hands the tokens back as a linked output (a view of the same memory): the expert path's
        # gradient of the tokens then reaches the router's backward, which adds it inside its dx kernel, so
        # x's gradient is formed in one pass instead of autograd adding the two paths' gradients afterwards
        # (the reference's autograd sums them, moe_layer.py L:288 and L:317-319)
        linked = self.router.take_linked_tokens()
        return self._experts_forward(flat if linked is None else linked, idx, weights).reshape(original_shape)

    @contextlib.contextmanager
    def _linked_tokens(self):
        r = self.router
        r._link_x = isinstance(r, MoERouter) and r.bias is None
        try:
            yield
        finally:
            r._link_x = False

    @contextlib.contextmanager
    def _deferred_router_check(self):
        """With ``check_numerics`` the router's checks (token conservation, non-finite logits) run at the end
        of the forward, at the synchronisation of the output NaN check, rather than right after the routing:
        the expert path is enqueued first, so the GPU does not wait for the host in the middle of the forward.
        The assertions and their order are the reference's (router first, then the output)."""
        r = self.router
        r._defer_check = self.check_numerics and r.sync_profile
        try:
            yield
        finally:
            r._defer_check = False

    def forward_normed(self, tokens: torch.Tensor, norm_weight: torch.Tensor, eps: float,
                       seq_offsets: Optional[torch.Tensor] = None,
                       token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``forward(rmsnorm(tokens))`` with the norm fused into the router's read of the hidden state
        (moe-engine/pkg/models/moe.py L:125-126): the normalised rows feed both the router and the experts."""
        original_shape = tokens.shape
        if tokens.dim() not in (2, 3):
            raise ValueError(f"tokens must be rank 2 or 3, got {tokens.dim()}")
        H = tokens.shape[-1]
        flat = tokens.reshape(-1, H)
        routed, seq = self._router_args(flat, original_shape, seq_offsets, token_mask)
        with self._deferred_router_check():
            xn, idx, weights, _cnt = self.router.forward_with_norm(routed, norm_weight, eps, **seq)
        return self._experts_forward(xn, idx, weights).reshape(original_shape)

    def _experts_forward(self, flat: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor,
                         mxfp4=None, int8=None) -> torch.Tensor:
        N = flat.shape[0]
        capacity = (
            math.ceil(self.capacity_factor * N * self.top_k / self.num_experts) if self.capacity_dropping else -1
        )
        p = ops.plan(idx, self.num_experts, capacity=capacity, layout=_LAYOUTS[self.layout])
        self.last_plan = p
        if mxfp4 is not None:
            train = torch.is_grad_enabled() and (flat.requires_grad or weights.requires_grad)
            timer = _ExpertTimer.new(flat)
            out = ExpertsMxfp4Fn.apply(flat, weights, *mxfp4, p, train, timer)
        elif int8 is not None:
            q, scale, wq, ws = int8
            timer = _ExpertTimer.new(flat)
            if timer is not None:
                timer.start()
            y = ops.swiglu_forward_int8(q, scale, wq, ws, p.offsets, row_slot=p.row_slot[:p.rows], top_k=self.top_k)
            if timer is not None:
                timer.stop()
            out = ops.combine(y, weights, p)
        elif self._fused():
            train = torch.is_grad_enabled() and any(
                t.requires_grad for t in (flat, weights, self.w_gate, self.w_up, self.w_down))
            timer = _ExpertTimer.new(flat)
            out = ExpertsFn.apply(flat, weights, self.w_gate, self.w_up, self.w_down, p, train, timer)
        else:
            timer = _ExpertTimer.new(flat)
            out = self._forward_per_expert(flat, weights, p, timer)
        self._expert_timer = timer
        if self.check_numerics:
            has_nan = torch.isnan(out).any()  # enqueued before the router's deferred checks synchronise
            self.router.check_pending()
            assert not has_nan, (
                "NaN detected in DistributedMoELayer output after combine step. "
                "Check expert FFN numerics and router weights."
            )
        return out

    # ------------------------------------------------------------------
    # fp8 (e4m3) forward, new: an inference variant of the fused expert path
    # ------------------------------------------------------------------
    def quantize_fp8(self):
        """e4m3 copies of the expert weights with one fp32 scale per weight row (per output channel), made
        on the GPU; kept until the weights change (their in-place version counters are checked)."""
        key = tuple((t.data_ptr(), t._version) for t in (self.w_gate, self.w_up, self.w_down))
        cache = getattr(self, "_fp8_cache", None)
        if cache is None or cache[0] != key:
            with torch.no_grad():
                q = [ops.quant_rows_fp8(t.detach()) for t in (self.w_gate, self.w_up, self.w_down)]
            self._fp8_cache = (key, tuple(t for t, _ in q), tuple(sc for _, sc in q))
        return self._fp8_cache[1], self._fp8_cache[2]

    @torch.no_grad()
    def forward_fp8(self, tokens: torch.Tensor, seq_offsets: Optional[torch.Tensor] = None,
                    token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The layer's forward with an e4m3 dispatch payload and e4m3 expert GEMMs (no autograd): router and
        planner as in ``forward``, the permute writes each token row quantized (one fp32 scale per row),
        the gate/up and down projections run on the fp8 MFMA with per-row x per-channel scales, the
        SwiGLU activations are quantized per row between them, and the combine is the bf16 one.  Needs
        the fused bf16 expert layout (``self._fused()``) and hidden_dim % 16 == 0.  ``seq_offsets`` and ``token_mask`` as in
        :meth:`forward`."""
        shape = tokens.shape
        return self._forward_fp8(tokens.reshape(-1, shape[-1]), shape, seq_offsets, token_mask).reshape(shape)

    def _forward_fp8(self, flat, shape, seq_offsets, token_mask, quantized=None):
        """``quantized``: the rows in e4m3 with their scales, where something before the layer has made them."""
        if not self._fused() or self.w_gate.dtype != torch.bfloat16:
            raise NotImplementedError("forward_fp8 needs the built-in SwiGLU experts in bfloat16")
        routed, seq = self._router_args(flat, shape, seq_offsets, token_mask)
        idx, weights, _cnt = self.router(routed, **seq)
        N = flat.shape[0]
        capacity = (
            math.ceil(self.capacity_factor * N * self.top_k / self.num_experts) if self.capacity_dropping else -1
        )
        p = ops.plan(idx, self.num_experts, capacity=capacity, layout=_LAYOUTS[self.layout])
        self.last_plan = p
        wq, ws = self.quantize_fp8()
        if quantized is None:
            xq, sx = ops.permute_fp8(flat, p)
        else:
            q, scale = quantized
            xq = ops.permute(q, p)
            sx = scale[p.row_slot[:p.rows] // self.top_k]  # (rows that no slot has: -1, any scale)
        _act, _hgu, y = ops.swiglu_forward_fp8(xq, sx, wq, ws, p.offsets, keep_preact=False)
        return ops.combine(y, weights, p)

    # ------------------------------------------------------------------
    # experts held in 4 bits (MXFP4), new: serving, and training around frozen experts
    # ------------------------------------------------------------------
    @torch.no_grad()
    def quantize_mxfp4(self):
        """Quantize the expert weights to MXFP4 (:func:`moe_mi355.ops.quant_mxfp4`: 4-bit e2m1 values, one power-of-two scale
        per 32 along the reduction) for :meth:`forward_mxfp4`, on the GPU.  The quantized weights stay as they are until this
        is called again, whatever becomes of the parameters, and move with the layer.  Returns ``((gate, up, down), (their
        scales))``, for :meth:`load_mxfp4` to take again: they are not in the layer's ``state_dict``."""
        if any(t is None for t in (self.w_gate, self.w_up, self.w_down)):
            raise RuntimeError("quantize_mxfp4: the layer's full-width weights were dropped")
        if self.w_gate.shape[-1] % ops.MXFP4_BLOCK or self.w_gate.shape[1] % ops.MXFP4_BLOCK:
            raise NotImplementedError(f"quantize_mxfp4 needs hidden and ffn dims that are multiples of {ops.MXFP4_BLOCK}")
        q = [ops.quant_mxfp4(t.detach()) for t in (self.w_gate, self.w_up, self.w_down)]
        return self.load_mxfp4([t for t, _ in q], [s for _, s in q])

    def load_mxfp4(self, weights, scales):
        """Take ``(gate, up, down)`` and their scales for :meth:`forward_mxfp4`: what :meth:`quantize_mxfp4` returned, or
        weights quantized elsewhere to the layout of :func:`moe_mi355.ops.quant_mxfp4` ([E, F, H / 2], [E, F, H / 2] and
        [E, H, F / 2] bytes; the last dims of the scales H / 32, H / 32 and F / 32).  They are kept as they are, on the router's
        device.  A layer that only serves them may drop its full-width parameters (``layer.w_gate = layer.w_up =
        layer.w_down = None``).  Returns them."""
        wq, ws, F_ = ops.mxfp4_weights("load_mxfp4", weights, scales, self.hidden_dim)
        if wq[0].shape[0] != len(self.local_expert_ids) or F_ != self.ffn_dim:
            raise ValueError(f"load_mxfp4: the layer has {len(self.local_expert_ids)} experts of ffn_dim {self.ffn_dim}, got "
                             f"{wq[0].shape[0]} of {F_}")
        dev = self.router.gate_w.device
        with torch.inference_mode(False):  # tensors of inference mode could not be saved for a backward
            for name, t in zip(_MXFP4, wq + ws):
                setattr(self, name, (t.clone() if t.is_inference() else t.detach()).to(dev))
        return self._mxfp4_weights()

    def _mxfp4_weights(self):
        q = tuple(getattr(self, name) for name in _MXFP4)
        return q[:3], q[3:]

    def forward_mxfp4(self, tokens: torch.Tensor, seq_offsets: Optional[torch.Tensor] = None,
                      token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``forward`` with the experts' weights as :meth:`quantize_mxfp4` or :meth:`load_mxfp4` left them: bf16 rows, 4-bit
        weights, from one decoded token to a long prefill.  Differentiable in the tokens and the router; the 4-bit weights are constants (the
        layer's own expert parameters get no gradient), so a router, or what lies before the layer, can be trained around
        experts in the form that they are served in.  Needs the built-in SwiGLU experts and bfloat16 tokens."""
        q = self._mxfp4_weights()
        if q[0][0] is None:
            raise RuntimeError("forward_mxfp4: call quantize_mxfp4() or load_mxfp4() first")
        if not all(type(m) is _SwiGLUExpert and m.w_gate._owner() is self for m in self.experts):
            raise NotImplementedError("forward_mxfp4 needs the built-in SwiGLU experts")
        if tokens.dim() not in (2, 3):
            raise ValueError(f"tokens must be rank 2 or 3, got {tokens.dim()}")
        if tokens.dtype != torch.bfloat16:
            raise TypeError(f"forward_mxfp4 takes bfloat16 tokens, got {tokens.dtype}")
        flat = tokens.reshape(-1, tokens.shape[-1])
        routed, seq = self._router_args(flat, tokens.shape, seq_offsets, token_mask)
        with self._deferred_router_check(), self._linked_tokens():
            idx, weights, _cnt = self.router(routed, **seq)
        linked = self.router.take_linked_tokens()
        return self._experts_forward(flat if linked is None else linked, idx, weights, q).reshape(tokens.shape)

    # ------------------------------------------------------------------
    # experts held in int8, new: serving
    # ------------------------------------------------------------------
    @torch.no_grad()
    def quantize_int8(self):
        """Quantize the expert weights to int8 with one fp32 scale per output channel (:func:`moe_mi355.ops.quant_rows_int8`)
        for :meth:`forward_int8`, on the GPU.  As :meth:`quantize_mxfp4`: they stay as they are until this is called again, move
        with the layer and are not in its ``state_dict``.  Returns ``((gate, up, down), (their scales))``."""
        if any(t is None for t in (self.w_gate, self.w_up, self.w_down)):
            raise RuntimeError("quantize_int8: the layer's full-width weights were dropped")
        if self.w_gate.shape[-1] % 16 or self.w_gate.shape[1] % 16:
            raise NotImplementedError("quantize_int8 needs hidden and ffn dims that are multiples of 16")
        q = [ops.quant_rows_int8(t.detach()) for t in (self.w_gate, self.w_up, self.w_down)]
        return self.load_int8([t for t, _ in q], [s for _, s in q])

    def load_int8(self, weights, scales):
        """Take ``(gate, up, down)`` and their scales for :meth:`forward_int8`: what :meth:`quantize_int8` returned, or weights
        quantized elsewhere (int8 [E, F, H], [E, F, H] and [E, H, F]; float32 [E, F], [E, F] and [E, H]).  They are kept as they
        are, on the router's device.  A layer that only serves them may drop its full-width parameters.  Returns them."""
        weights, scales = list(weights), list(scales)
        if len(weights) != 3 or len(scales) != 3:
            raise ValueError(f"load_int8: takes (gate, up, down) and three scales, got {len(weights)} and {len(scales)}")
        E, F_, H = len(self.local_expert_ids), self.ffn_dim, self.hidden_dim
        for name, w, s, shape in zip(("gate", "up", "down"), weights, scales, ((E, F_, H), (E, F_, H), (E, H, F_))):
            if w.dtype != torch.int8 or s.dtype != torch.float32:
                raise TypeError(f"load_int8: {name} must be int8 with float32 scales, got {w.dtype} and {s.dtype}")
            if tuple(w.shape) != shape or tuple(s.shape) != shape[:2]:
                raise ValueError(f"load_int8: {name} must be {list(shape)} with scales {list(shape[:2])}, got {list(w.shape)} and "
                                 f"{list(s.shape)}")
        dev = self.router.gate_w.device
        with torch.inference_mode(False):
            for name, t in zip(_INT8, [*weights, *scales]):
                t = t.clone() if t.is_inference() else t.detach()
                t = t.contiguous().to(dev)
                setattr(self, name, t.view(torch.int32) if t.dtype == torch.float32 else t)
        return self._int8_weights()

    def _int8_weights(self):
        q = tuple(getattr(self, name) for name in _INT8)
        return q[:3], tuple(None if t is None else t.view(torch.float32) for t in q[3:])

    @torch.no_grad()
    def forward_int8(self, tokens: torch.Tensor, seq_offsets: Optional[torch.Tensor] = None,
                     token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``forward`` for serving (no autograd) on the weights as :meth:`quantize_int8` or :meth:`load_int8` left them: router,
        planner and combine as in ``forward``; the tokens are quantized to int8 once, the experts read them through the plan,
        and the SwiGLU activations are quantized per row between the projections.  From one decoded token to a long prompt; a
        token's experts give the same bits in any batch.  Needs the built-in SwiGLU experts and bfloat16 tokens."""
        if tokens.dim() not in (2, 3):
            raise ValueError(f"tokens must be rank 2 or 3, got {tokens.dim()}")
        flat = tokens.reshape(-1, tokens.shape[-1])
        return self._forward_int8(flat, tokens.shape, seq_offsets, token_mask).reshape(tokens.shape)

    def _forward_int8(self, flat, shape, seq_offsets, token_mask, quantized=None):
        """``quantized``: the rows in int8 with their scales, where something before the layer has made them."""
        wq, ws = self._int8_weights()
        if wq[0] is None:
            raise RuntimeError("forward_int8: call quantize_int8() or load_int8() first")
        if not all(type(m) is _SwiGLUExpert and m.w_gate._owner() is self for m in self.experts):
            raise NotImplementedError("forward_int8 needs the built-in SwiGLU experts")
        if flat.dtype != torch.bfloat16:
            raise TypeError(f"forward_int8 takes bfloat16 tokens, got {flat.dtype}")
        q, scale = ops.quant_rows_int8(flat) if quantized is None else quantized
        routed, seq = self._router_args(flat, shape, seq_offsets, token_mask)
        with self._deferred_router_check():
            idx, weights, _cnt = self.router(routed, **seq)
        return self._experts_forward(flat, idx, weights, int8=(q, scale, wq, ws))

    def _forward_per_expert(self, flat: torch.Tensor, weights: torch.Tensor, p: ops.Plan,
                            timer: Optional["_ExpertTimer"] = None) -> torch.Tensor:
        """Dispatch/combine kernels around per-expert module calls (custom experts, non-bf16 dtypes)."""
        xp = PermuteFn.apply(flat, p)
        offs = p.offsets.tolist()  # segment bounds for the per-expert calls
        parts = []
        if timer is not None:
            timer.start()
        for i, expert in enumerate(self.experts):
            lo, hi = offs[i], offs[i + 1]
            if lo < hi:
                parts.append(expert(xp[lo:hi]))
        if timer is not None:
            timer.stop()
        tail = p.rows - offs[len(self.experts)]
        if tail > 0:
            parts.append(xp.new_zeros((tail, xp.shape[1])))
        y = torch.cat(parts, 0) if parts else xp.new_zeros(xp.shape)
        return CombineFn.apply(y.contiguous(), weights, p)

    def _expert_to_rank(self, expert_ids: torch.Tensor) -> torch.Tensor:
        """Every expert lives on this (single) rank (reference L:362-389 at ep_size=1)."""
        return torch.zeros_like(expert_ids, dtype=torch.long)
