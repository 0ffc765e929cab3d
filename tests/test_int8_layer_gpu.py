"""The layer and the block on int8 experts and with the residual's addition in the norm: forwards against the oracles, a stack's
training step against the same stack with the sums made outside, a stack served in int8 and e4m3 as it would be."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import ops
from oracle import int8 as OI
from oracle import norm as ON
from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer
from pkg.models import RMSNorm, ToyMoEBlock

pytestmark = pytest.mark.gpu

B = torch.bfloat16


def _gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def _layer(H, F, E, K, cls=DistributedMoELayer, dtype=B, **kw):
    torch.manual_seed(H + F + E)
    return cls(H, F, E, K, build_topology(), dtype=dtype, **kw).to(dev())


def _combined(layer, p, w, y, ty):
    """Each token's weighted sum of its live rows of y, and how far a bf16 one may be off."""
    N, K = w.shape
    used = int(p.offsets[-1])
    ref, tol = (torch.zeros(N, y.shape[1], dtype=torch.float64, device=dev()) for _ in range(2))
    for k in range(K):
        row = p.slot_row.long().reshape(N, K)[:, k]
        live = (row >= 0) & (row < used)
        if p.drop is not None:
            live &= ~p.drop[:, k]
        ref[live] += w[live, k].double().unsqueeze(1) * y[row[live]]
        tol[live] += w[live, k].double().unsqueeze(1) * (ty + 2.0 ** -22 * y.abs())[row[live]]
    return ref, tol + OI.BF16 * (ref.abs() + tol) + 1e-30


def _experts(layer, q, s, p):
    used = int(p.offsets[-1])
    token = p.row_slot[:used].long() // layer.top_k
    wq, ws = layer._int8_weights()
    return OI.swiglu_fwd(q[token], s[token], wq, ws, p.offsets.tolist())


@pytest.mark.parametrize("layout,drops", [("routed", False), ("reference", False), ("routed", True), ("reference", True)])
@pytest.mark.parametrize("N,H,F,E,K", [(1, 256, 512, 8, 2), (37, 128, 96, 4, 3), (600, 256, 384, 8, 2)])
def test_layer_forward(N, H, F, E, K, layout, drops):
    say(f"[int8 layer] N={N} H={H} F={F} E={E} K={K} {layout} drops={drops}")
    layer = _layer(H, F, E, K, layout=layout, capacity_dropping=drops, capacity_factor=1.0)
    x = torch.randn(N, H, device=dev(), generator=_gen(N)).to(B)
    with pytest.raises(RuntimeError, match="quantize_int8"):
        layer.forward_int8(x)
    wq, ws = layer.quantize_int8()
    for t, a, b in zip((layer.w_gate, layer.w_up, layer.w_down), wq, ws):
        rq, rs = OI.quant(t.detach())
        assert torch.equal(a, rq) and torch.equal(b, rs.float())
    out = layer.forward_int8(x)
    assert layer.last_expert_compute_ms >= 0.0
    with torch.no_grad():
        w = layer.router(x)[1]
    q, s = ops.quant_rows_int8(x)
    y, ty = _experts(layer, q, s, layer.last_plan)
    ref, tol = _combined(layer, layer.last_plan, w, y, ty)
    assert float(((out.double() - ref).abs() / tol).max()) <= 1.0
    assert torch.equal(layer.forward_int8(x.view(1, N, H))[0], out)
    # the weights stay what they were quantized from
    with torch.no_grad():
        layer.w_gate.zero_()
    assert torch.equal(layer.forward_int8(x), out)
    layer.quantize_int8()
    assert float(layer.forward_int8(x).abs().max()) == 0.0


def test_layer_without_its_full_width_weights_and_nothing_to_do():
    layer = _layer(128, 96, 4, 2, layout="routed")
    x = torch.randn(40, 128, device=dev(), generator=_gen(1)).to(B)
    layer.quantize_int8()
    want = layer.forward_int8(x)
    other = _layer(128, 96, 4, 2, layout="routed")
    other.load_state_dict(layer.state_dict())
    other.load_int8(*layer._int8_weights())
    other.w_gate = other.w_up = other.w_down = None
    assert torch.equal(other.forward_int8(x), want)
    assert layer.forward_int8(x[:0]).shape == (0, 128)


def test_layer_checks_its_numerics():
    layer = _layer(128, 96, 4, 2, layout="routed")
    layer.quantize_int8()
    x = torch.randn(8, 128, device=dev(), generator=_gen(1)).to(B)
    layer.int8_down_scale[:] = torch.tensor(float("nan")).view(torch.int32).item()
    with pytest.raises(AssertionError, match="NaN"):
        layer.forward_int8(x)


@pytest.mark.parametrize("dtype", [B, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(1, 64), (33, 2048), (4, 6, 128)], ids=str)
def test_norm_module(shape, dtype):
    torch.manual_seed(0)
    H = shape[-1]
    norm = RMSNorm(H).to(dev())
    with torch.no_grad():
        norm.weight.add_(0.1 * torch.randn(H, device=dev()))
    x, r, gx, gh = (torch.randn(shape, device=dev(), generator=_gen(i)).to(dtype) for i in range(4))
    x.requires_grad_()
    r.requires_grad_()
    xn, h = norm(x, residual=r)
    assert xn.shape == h.shape == shape and torch.equal(h, (x + r).detach()) and torch.equal(xn, norm(h.detach()))
    torch.autograd.backward([xn, h], [gx, gh])
    assert torch.equal(x.grad, r.grad)
    d, dw = ON.rmsnorm_residual_bwd(h.detach().reshape(-1, H), norm.weight.detach(), gx.reshape(-1, H), gh.reshape(-1, H), norm.eps)
    step = OI.BF16 if dtype == B else 1e-5
    scale = d.abs().amax()
    assert float((x.grad.reshape(-1, H).double() - d).abs().max()) <= float(scale) * step
    assert float((norm.weight.grad.double() - dw).abs().max()) <= float(dw.abs().amax()) * 1e-5
    # only one of the outputs used, only one of the inputs trained, a residual that is its own input
    x.grad = r.grad = None
    norm(x, residual=r.detach())[0].backward(gx)
    only = x.grad.clone()
    x.grad = None
    norm(x.detach(), residual=r)[0].backward(gx)
    assert torch.equal(only, r.grad)
    x.grad = None
    y, h = norm(x, residual=x)
    (y * gx).sum().backward()
    with torch.no_grad():
        ref = ON.rmsnorm_bwd((x + x).reshape(-1, H), norm.weight, gx.reshape(-1, H), norm.eps)[0] * 2
    # two bf16 gradients are added and rounded once more
    assert float((x.grad.reshape(-1, H).double() - ref).abs().max()) <= float(ref.abs().amax()) * 2 * step


def _stack(n, H, F, E, K, dtype, **kw):
    torch.manual_seed(7)
    blocks = [ToyMoEBlock(H, F, E, K, build_topology(), dtype=dtype, layout="routed", check_numerics=False, **kw).to(dev())
              for _ in range(n)]
    return blocks, RMSNorm(H).to(dev())


def test_a_stack_trains_as_with_the_sums_outside():
    """fp32: a stack whose sums are inside the norms against the same stack with the sums made by torch; every gradient."""
    H, F, E, K = 128, 96, 4, 2
    blocks, last = _stack(3, H, F, E, K, torch.float32)
    x0 = torch.randn(2, 50, H, device=dev(), generator=_gen(3))
    g = torch.randn(2, 50, H, device=dev(), generator=_gen(4))
    params = [p for m in (*blocks, last) for p in m.parameters()]

    def grads(run):
        x = x0.clone().requires_grad_()
        out = run(x)
        return out.detach(), torch.autograd.grad(out, [x, *params], g)

    def inside(x):
        out, h = torch.zeros_like(x), x
        for b in blocks:
            out, h = b(out, residual=h)
        return last(out, residual=h)[0]

    def outside(x):
        for b in blocks:
            x = x + b.moe(b.norm(x))
        return last(x)

    a, ga = grads(inside)
    b, gb = grads(outside)
    assert torch.equal(a, b)
    for u, v in zip(ga, gb):
        # the same products; sums of gradients in another order
        assert float((u - v).abs().max()) <= 1e-5 * max(float(v.abs().max()), 1e-6)


def test_a_captured_training_step_of_a_stack():
    H, F, E, K = 128, 96, 4, 2
    blocks, last = _stack(2, H, F, E, K, B)
    for b in blocks:
        b.moe.router.sync_profile = False
    x = torch.randn(64, H, device=dev(), generator=_gen(3)).to(B)
    params = [p for m in (*blocks, last) for p in m.parameters()]

    def step():
        out, h = blocks[0](x, residual=x * 0.5)
        out, h = blocks[1](out, residual=h)
        y = last(out, residual=h)[0]
        return [y, *torch.autograd.grad(y.float().square().sum(), params)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = step()
        for i in range(3):
            x.copy_(torch.randn(64, H, device=dev(), generator=_gen(30 + i)).to(B))
            g.replay()
            stream.synchronize()
            want = step()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {i}"
    torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("N", [1, 5, 300])
def test_a_stack_served_in_8_bits(N, fmt):
    H, F, E, K = 256, 384, 8, 2
    blocks, last = _stack(2, H, F, E, K, B)
    x = torch.randn(N, H, device=dev(), generator=_gen(N)).to(B)
    with torch.no_grad():
        for b in blocks:
            b.norm.weight.add_(0.1 * torch.randn(H, device=dev(), generator=_gen(5)))
            if fmt == "int8":
                b.moe.quantize_int8()
    serve = (lambda b, *a, **k: b.forward_int8(*a, **k)) if fmt == "int8" else (lambda b, *a, **k: b.forward_fp8(*a, **k))
    out, h = serve(blocks[0], x, residual=x * 0.5)
    rh = x + x * 0.5
    assert torch.equal(h, rh)
    out2, h2 = serve(blocks[1], out, residual=h)
    assert torch.equal(h2, out + h)
    y = last(out2, residual=h2)[0]
    # without a residual the block adds its input itself: the same rows, so the same bits
    alone = serve(blocks[0], rh)
    assert torch.equal(alone, rh + out)
    assert torch.equal(serve(blocks[0], rh.view(1, N, H))[0], alone)
    if fmt == "int8":
        p = blocks[1].moe.last_plan  # of the last call, block 1's
        q, s, xn, _ = ops.rmsnorm_quant(out, blocks[1].norm.weight, blocks[1].norm.eps, residual=h, keep_norm=True)
        with torch.no_grad():
            w = blocks[1].moe.router(xn)[1]
        ref, tol = _combined(blocks[1].moe, p, w, *_experts(blocks[1].moe, q, s, p))
        assert float(((out2.double() - ref).abs() / tol).max()) <= 1.0
        # a token's experts give the same bits alone as in its batch
        if N > 1:
            rows = torch.cat([blocks[0].forward_int8(x[i:i + 1], residual=x[i:i + 1] * 0.5)[0] for i in range(0, N, 37)])
            with torch.no_grad():
                xr = blocks[0].norm.quantized(x, x * 0.5)[2]
                same = (blocks[0].moe.router(xr)[1] == torch.cat([blocks[0].moe.router(xr[i:i + 1])[1] for i in range(N)])).all(-1)
            assert torch.equal(rows[same[::37]], out[::37][same[::37]])
    # near the bf16 block: every factor is off by at most a few hundredths of its row's largest
    with torch.no_grad():
        plain = blocks[0](x, residual=x * 0.5)[0]
    assert float((out - plain).float().abs().max()) <= 0.1 * float(plain.float().abs().max())
    assert bool(torch.isfinite(y).all())


def test_served_and_captured():
    H, F, E, K = 256, 128, 8, 2
    blocks, _ = _stack(1, H, F, E, K, B)
    block = blocks[0]
    block.moe.quantize_int8()
    block.moe.router.sync_profile = False
    x = torch.randn(6, H, device=dev(), generator=_gen(1)).to(B)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.no_grad():
        for _ in range(2):
            block.forward_int8(x, residual=x)
            block.forward_fp8(x, residual=x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = (*block.forward_int8(x, residual=x), *block.forward_fp8(x, residual=x))
        for i in range(3):
            x.copy_(torch.randn(6, H, device=dev(), generator=_gen(20 + i)).to(B))
            g.replay()
            stream.synchronize()
            want = (*block.forward_int8(x, residual=x), *block.forward_fp8(x, residual=x))
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {i}"
    torch.cuda.current_stream().wait_stream(stream)


def test_sequences_and_masks_pass_through():
    H, F, E, K = 128, 96, 4, 2
    blocks, _ = _stack(1, H, F, E, K, B, seq_balance_coef=0.01)
    block = blocks[0]
    block.moe.quantize_int8()
    x = torch.randn(3, 20, H, device=dev(), generator=_gen(1)).to(B)
    mask = torch.rand(3, 20, device=dev(), generator=_gen(2)) < 0.7
    losses = []
    for call in (block.forward_int8, block.forward_fp8, lambda *a, **k: block(*a, **k)):
        with torch.no_grad():
            call(x, residual=x, token_mask=mask)
            losses.append(float(block.moe.router.last_seq_balance_loss))
    assert losses[0] == losses[1] == losses[2] > 0.0


def _block(H, F, E, K, layout, drops):
    torch.manual_seed(11)
    block = ToyMoEBlock(H, F, E, K, build_topology(), dtype=B, layout=layout, capacity_dropping=drops, capacity_factor=1.0,
                        check_numerics=False).to(dev())
    with torch.no_grad():
        block.norm.weight.add_(0.1 * torch.randn(H, device=dev(), generator=_gen(5)))
    return block


LAYOUTS = [("routed", False), ("reference", False), ("routed", True), ("reference", True)]


@pytest.mark.parametrize("layout,drops", LAYOUTS)
@pytest.mark.parametrize("N", [1, 37, 600])
def test_block_in_e4m3_is_its_parts(N, layout, drops):
    """The block on the norm's e4m3 rows: each slot's row and scale placed where the plan says, the experts' products and the
    combine, bit for bit.  Every row has a largest value, and so a scale, of its own: another row's would show."""
    H, F, E, K = 256, 384, 8, 2
    say(f"[block e4m3] N={N} {layout} drops={drops}")
    block = _block(H, F, E, K, layout, drops)
    x = torch.randn(N, H, device=dev(), generator=_gen(N)).to(B)
    r = torch.randn(N, H, device=dev(), generator=_gen(N + 1)).to(B)
    r[:, 0] += torch.exp2(torch.arange(N, device=dev()) % 9.0).to(B) * 4  # the largest of a row by another factor each
    out, h = block.forward_fp8(x, residual=r)
    p = block.moe.last_plan
    q, s, xn, hq = ops.rmsnorm_quant(x, block.norm.weight, block.norm.eps, residual=r, fmt="e4m3", keep_norm=True)
    assert torch.equal(h, hq)
    with torch.no_grad():
        w = block.moe.router(xn)[1]
    row = p.slot_row.long().reshape(N, K)
    used = int(p.offsets[-1])
    xq, sx = torch.zeros(p.rows, H, dtype=torch.uint8, device=dev()), torch.ones(p.rows, device=dev())
    for k in range(K):
        live = (row[:, k] >= 0) & (row[:, k] < used)
        xq[row[live, k]], sx[row[live, k]] = q[live], s[live]
    if drops and N > 1:
        assert bool(p.drop.any()) if p.drop is not None else used < N * K
    wq, ws = block.moe.quantize_fp8()
    y = ops.swiglu_forward_fp8(xq, sx, wq, ws, p.offsets, keep_preact=False)[2]
    want = ops.combine(y, w, p)
    assert torch.equal(out, want)
    if N >= 37:
        assert len(s.unique()) >= 9  # rows that differ


@pytest.mark.parametrize("layout,drops", LAYOUTS)
@pytest.mark.parametrize("N", [1, 37, 600])
def test_block_in_int8_with_layouts_and_drops(N, layout, drops):
    H, F, E, K = 256, 384, 8, 2
    say(f"[block int8] N={N} {layout} drops={drops}")
    block = _block(H, F, E, K, layout, drops)
    block.moe.quantize_int8()
    x = torch.randn(N, H, device=dev(), generator=_gen(N)).to(B)
    r = torch.randn(N, H, device=dev(), generator=_gen(N + 1)).to(B)
    r[:, 0] += torch.exp2(torch.arange(N, device=dev()) % 9.0).to(B) * 4
    out, h = block.forward_int8(x, residual=r)
    p = block.moe.last_plan
    q, s, xn, hq = ops.rmsnorm_quant(x, block.norm.weight, block.norm.eps, residual=r, keep_norm=True)
    assert torch.equal(h, hq)
    with torch.no_grad():
        w = block.moe.router(xn)[1]
    ref, tol = _combined(block.moe, p, w, *_experts(block.moe, q, s, p))
    assert float(((out.double() - ref).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("dtype", [B, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64), (2, 1, 5, 528)], ids=str)
def test_gradients_accumulate_apart(shape, dtype):
    """x and the residual have one gradient; as leaves each keeps its own, and a second backward adds to each once."""
    norm = RMSNorm(shape[-1]).to(dev())
    x, r, gx, gh = (torch.randn(shape, device=dev(), generator=_gen(i)).to(dtype) for i in range(4))
    for run in (lambda a, b: norm(a, residual=b), lambda a, b: norm(a, residual=b)[1:], lambda a, b: norm(a, residual=b)[:1]):
        x, r = x.detach().requires_grad_(), r.detach().requires_grad_()
        outs = run(x, r)
        once = torch.autograd.grad(outs, [x, r], ([gx, gh] if len(outs) == 2 else [gx]))
        assert torch.equal(once[0], once[1])
        for _ in range(2):
            outs = run(x, r)
            torch.autograd.backward(outs, [gx, gh] if len(outs) == 2 else [gx])
        assert x.grad.untyped_storage().data_ptr() != r.grad.untyped_storage().data_ptr()
        assert torch.equal(x.grad, once[0] + once[0]) and torch.equal(r.grad, once[0] + once[0])
        x.grad.zero_()
        assert torch.equal(r.grad, once[0] + once[0])


def test_a_blocks_gradients_accumulate_apart():
    blocks, _ = _stack(1, 128, 96, 4, 2, torch.float32)
    x, r = (torch.randn(2, 20, 128, device=dev(), generator=_gen(i)).requires_grad_() for i in range(2))
    g = torch.randn(2, 20, 128, device=dev(), generator=_gen(3))
    once = torch.autograd.grad(blocks[0](x, residual=r), [x, r], [g, g])
    for _ in range(2):
        torch.autograd.backward(blocks[0](x, residual=r), [g, g])
    for t in (x, r):
        assert float((t.grad - 2 * once[0]).abs().max()) <= 1e-5 * float(once[0].abs().max())


@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64)], ids=str)
def test_outputs_written_in_place(shape):
    """The normalised rows may be written in place; writing the sum, which the backward reads, is noticed."""
    norm = RMSNorm(shape[-1]).to(dev())
    x, r, g = (torch.randn(shape, device=dev(), generator=_gen(i)) for i in range(3))
    x.requires_grad_()
    want = torch.autograd.grad(norm(x, residual=r)[0], x, 3 * g)[0]
    y = norm(x, residual=r)[0].mul_(3)
    assert torch.equal(torch.autograd.grad(y, x, g)[0], want)
    y, h = norm(x, residual=r)
    h.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward(g)
