"""The MoE layer on 4-bit experts: its forward against the oracle's experts on the dequantized weights, its gradients against
the same layer in bf16 on those weights, and a router trained with the balance loss of sequences around frozen 4-bit experts,
then served with them."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import ops
from oracle import mxfp4 as OX
from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer

pytestmark = pytest.mark.gpu

B = torch.bfloat16


def _layer(H, F, E, K, **kw):
    torch.manual_seed(H + F + E)
    return DistributedMoELayer(H, F, E, K, build_topology(), dtype=B, **kw).to(dev())


@pytest.mark.parametrize("layout,drops", [("routed", False), ("reference", False), ("routed", True)])
@pytest.mark.parametrize("N,H,F,E,K", [(1, 256, 512, 8, 2), (37, 128, 96, 4, 3), (600, 256, 384, 8, 2)])
def test_forward(N, H, F, E, K, layout, drops):
    say(f"[mxfp4 layer] N={N} H={H} F={F} E={E} K={K} {layout} drops={drops}")
    layer = _layer(H, F, E, K, layout=layout, capacity_dropping=drops, capacity_factor=1.0)
    x = torch.randn(N, H, device=dev(), generator=torch.Generator(device=dev()).manual_seed(N)).to(B)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="quantize_mxfp4"):
            layer.forward_mxfp4(x)
        q, s = layer.quantize_mxfp4()
        out = layer.forward_mxfp4(x)
        w = layer.router(x)[1]
    p = layer.last_plan
    xp = ops.permute(x, p)
    used = int(p.offsets[-1])
    _, y, _, ty = OX.swiglu_fwd(xp[:used], [OX.dequant(a, b) for a, b in zip(q, s)], p.offsets.tolist())
    ref, tol = (torch.zeros(N, H, dtype=torch.float64, device=dev()) for _ in range(2))
    for k in range(K):
        row = p.slot_row.long().reshape(N, K)[:, k]
        live = (row >= 0) & (row < used)
        if p.drop is not None:
            live &= ~p.drop[:, k]
        ref[live] += w[live, k].double().unsqueeze(1) * y[row[live]]
        tol[live] += w[live, k].double().unsqueeze(1) * (ty + 2.0 ** -22 * y.abs())[row[live]]
    tol = tol + 2.0 ** -8 * (ref.abs() + tol) + 1e-30
    assert float(((out.double() - ref).abs() / tol).max()) <= 1.0
    # the weights stay what they were quantized from
    with torch.no_grad():
        layer.w_gate.zero_()
        assert torch.equal(layer.forward_mxfp4(x), out)
        layer.quantize_mxfp4()
        assert float(layer.forward_mxfp4(x).abs().max()) == 0.0


@pytest.mark.parametrize("N,H,F,E,K", [(5, 128, 160, 4, 2), (700, 256, 512, 8, 2)])
def test_gradients(N, H, F, E, K):
    """Tokens and gate, against the bf16 layer whose experts hold the dequantized weights (exact in bf16).  The two paths round
    differently in two places (g and u are rounded before act there), so each gradient is within a few roundings, 2^-8 each,
    in norm."""
    say(f"[mxfp4 layer gradients] N={N} H={H} F={F}")
    layer = _layer(H, F, E, K, layout="routed")
    with torch.no_grad():
        q, s = layer.quantize_mxfp4()
        for p, a, b in zip((layer.w_gate, layer.w_up, layer.w_down), q, s):
            p.copy_(ops.dequant_mxfp4(a, b))
    x = torch.randn(N, H, device=dev()).to(B).requires_grad_(True)
    gout = torch.randn(N, H, device=dev()).to(B)
    a = torch.autograd.grad(layer.forward_mxfp4(x), [x, layer.router.gate_w], gout)
    b = torch.autograd.grad(layer(x), [x, layer.router.gate_w], gout)
    for u, v in zip(a, b):
        assert float((u.double() - v.double()).norm() / v.double().norm()) <= 6 * 2.0 ** -8
    out = layer.forward_mxfp4(x)
    assert out.requires_grad
    got = torch.autograd.grad(out, [layer.w_gate, layer.w_up, layer.w_down], gout, allow_unused=True)
    assert all(g is None for g in got)


def test_train_the_router_around_frozen_experts_then_serve():
    """As they would be used together: padded batches through forward_mxfp4 with the balance loss of sequences, gate updates,
    then decoding token by token; the decoded rows have the bits of the batch's."""
    say("[mxfp4 train + serve]")
    Bn, S, H, F, E, K = 4, 24, 256, 512, 8, 2
    layer = _layer(H, F, E, K, layout="routed", seq_balance_coef=1.0, z_loss_coef=1e-3)
    layer.quantize_mxfp4()
    gate = layer.router.gate_w
    lengths = torch.tensor([[24], [3], [0], [17]], device=dev())
    mask = torch.arange(S, device=dev()) < lengths
    for step in range(3):
        g = torch.Generator(device=dev()).manual_seed(step)
        x = torch.randn(Bn, S, H, device=dev(), generator=g).to(B)
        before = gate.detach().clone()
        out = layer.forward_mxfp4(x, token_mask=mask)
        r = layer.router
        assert r.last_seq_tokens.tolist() == [24, 3, 0, 17, 44, 3] and int(r.last_seq_counts.sum()) == 44 * K
        loss = (out.float() ** 2)[mask].mean() + r.last_seq_balance_loss + r.last_z_loss
        gate.grad = None
        loss.backward()
        assert bool(torch.isfinite(gate.grad).all()) and float(gate.grad.abs().max()) > 0
        assert layer.w_gate.grad is None and layer.w_down.grad is None
        with torch.no_grad():
            gate -= (0.1 * gate.grad.float()).to(B)
        assert not torch.equal(gate, before)
    with torch.no_grad():
        x = torch.randn(16, H, device=dev()).to(B)
        whole = layer.forward_mxfp4(x)
        for t in range(16):
            assert torch.equal(layer.forward_mxfp4(x[t:t + 1]), whole[t:t + 1])


def test_decode_graph():
    say("[mxfp4 decode graph]")
    layer = _layer(512, 768, 16, 4, layout="routed", check_numerics=False)
    layer.quantize_mxfp4()
    x = torch.randn(6, 512, device=dev()).to(B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            buf = x.clone()
            layer.forward_mxfp4(buf)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = layer.forward_mxfp4(buf)
        for i in range(4):
            buf.copy_(torch.randn(6, 512, device=dev()).to(B))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, layer.forward_mxfp4(buf)), i


def test_training_step_graph():
    """A training step of the router and the tokens around 4-bit experts, captured and replayed."""
    say("[mxfp4 training graph]")
    from test_graph_gpu import _replays_match_eager

    layer = _layer(256, 512, 8, 2, layout="routed", check_numerics=False, seq_balance_coef=0.5, z_loss_coef=1e-3)
    layer.quantize_mxfp4()
    x = torch.randn(6, 50, 256, device=dev()).to(B).requires_grad_(True)
    mask = torch.arange(50, device=dev()) < torch.tensor([[50], [3], [0], [17], [49], [1]], device=dev())
    gout, one = torch.randn(6, 50, 256, device=dev()).to(B), torch.ones((), device=dev())
    gate = layer.router.gate_w

    def step():
        out = layer.forward_mxfp4(x, token_mask=mask)
        r = layer.router
        bal, z = r.last_seq_balance_loss, r.last_z_loss
        dx, dg = torch.autograd.grad((out, bal, z), (x, gate), grad_outputs=(gout, one, one))
        res = out.detach(), bal.detach(), z.detach(), r.last_seq_counts, r.last_seq_tokens, dx, dg
        # the layer keeps its last losses; drop them, and with them the step's autograd graph
        r.last_seq_balance_loss = r.last_z_loss = r.last_aux_loss = None
        return res

    _replays_match_eager(step, ("out", "balance", "z", "counts", "tokens", "dx", "dgate"))


def test_refusals():
    layer = _layer(64, 64, 4, 2)
    layer.quantize_mxfp4()
    with pytest.raises(TypeError):
        layer.forward_mxfp4(torch.randn(4, 64, device=dev()))
    with pytest.raises(ValueError):
        layer.forward_mxfp4(torch.randn(64, device=dev()).to(B))
    layer.experts = torch.nn.ModuleList([torch.nn.Linear(64, 64) for _ in range(4)])
    with pytest.raises(NotImplementedError):
        layer.forward_mxfp4(torch.randn(4, 64, device=dev()).to(B))
    with pytest.raises(NotImplementedError):
        _layer(48, 64, 4, 2).quantize_mxfp4()
