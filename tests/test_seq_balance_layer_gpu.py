"""The balance loss of sequences through the router, the layer and the block: its gradient joins dL/dlogits inside every form
of the router's backward, within bounds counted from the roundings (dL/dlogits to bf16 with bf16 tokens: 2^-8 of a term; the
outputs: 2^-8 of the value; fp32 sums of n terms: n 2^-24 of their magnitudes; dL/dlogits itself (3 E + 120) 2^-24 of its
terms' magnitudes)."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import ops
from moe_mi355.balance import balance_loss
from moe_mi355.norm import NormRouterCore
from moe_mi355.router import RouterCore
from oracle import balance as OB
from oracle import router as OR
from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer
from pkg.kernels.moe_router import MoERouter
from pkg.models import ToyMoEBlock

pytestmark = pytest.mark.gpu

B, F = torch.bfloat16, torch.float32
U = 2.0 ** -24
BC, ZC = 0.05, 1e-2

# (N, H, E, K, dtype): streaming (E <= 16, <= 32), wide (<= 64, <= 128), past it, fp32 in registers, fp32 matrix, generic
SHAPES = [(300, 256, 8, 2, B), (77, 1024, 8, 2, B), (130, 264, 24, 5, B), (200, 256, 64, 6, B), (90, 128, 128, 8, B),
          (60, 64, 200, 4, B), (120, 128, 8, 2, F), (100, 64, 64, 4, F), (70, 68, 18, 3, F)]
IDS = [f"N{s[0]}-H{s[1]}-E{s[2]}-K{s[3]}-{str(s[4])[6:]}" for s in SHAPES]


def _inputs(N, H, E, K, dt, seed=0):
    g = torch.Generator().manual_seed(N + H + E + seed)
    x = torch.randn(N, H, generator=g).to(dt)
    w = (torch.randn(H, E, generator=g) * H ** -0.5).to(dt)
    cuts = sorted(torch.randint(0, N + 1, (4,), generator=g).tolist())
    offs = torch.tensor([0] + cuts[:3] + [max(cuts[3], N - 5)])
    mask = torch.rand(N, generator=g) < 0.8
    return x, w, offs, mask


def _magnitude(ref, logits, offs, mask, K, E):
    """Magnitudes of the terms of dL/dlogits."""
    m = torch.zeros(logits.shape, dtype=torch.float64)
    n_all, used = max(1, int(ref["tokens"][-2])), max(1, int(ref["tokens"][-1]))
    for s in range(len(offs) - 1):
        t = torch.arange(int(offs[s]), int(offs[s + 1]))
        t = t[mask[t]]
        if len(t) == 0:
            continue
        f = E * ref["counts"][s].double() / (K * len(t))
        p = torch.softmax(logits[t].double(), 1)
        lse = torch.logsumexp(logits[t].double(), 1, keepdim=True)
        m[t] = p * (BC / (used * len(t)) * (f + (p * f).sum(1, keepdim=True)) + 2 * ZC / n_all * lse.abs())
    return m


def _check(got, G, mag, left, right, bf16, n, what):
    """got against left^T-style product G @ right (given as a function), within the bound."""
    E = G.shape[1]
    want, room = right(G), right(mag, True)
    tol = ((3 * E + 120) * U + (2.0 ** -8 if bf16 else 0.0) + (n + 2) * U) * room
    tol = tol + (2.0 ** -8 if bf16 else U) * (want.abs() + tol) + 1e-30
    off = ((got.detach().cpu().double() - want).abs() / tol).max()
    assert float(off) <= 1.0, f"{what}: {float(off):.3f} of the bound"


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_gradient_through_the_router(shape):
    N, H, E, K, dt = shape
    say(f"[seq balance router] {shape}")
    x, w, offs, mask = _inputs(*shape)
    xd, wd = (t.to(dev()).requires_grad_(True) for t in (x, w))
    idx, _w, _aux, _z, logits, _cnt, _st = RouterCore.apply(xd, wd, K, 0.0, 0.0, None, diff_logits=True)
    bal, z, counts, tokens, _ = balance_loss(logits, idx, offs.to(dev()), mask.to(dev()), BC, ZC)
    dx, dw = torch.autograd.grad(bal + z, (xd, wd))
    lg = logits.detach().cpu()
    ref = OB.balance(lg, idx.cpu(), offs, mask, BC, ZC)
    assert torch.equal(counts.cpu(), ref["counts"]) and torch.equal(tokens.cpu(), ref["tokens"])
    mag = _magnitude(ref, lg, offs, mask, K, E)
    X, W = x.double(), w.double()
    _check(dx, ref["dlogits"], mag, None, lambda g, a=False: g @ (W.abs() if a else W).T, dt == B, E, "dx")
    _check(dw, ref["dlogits"], mag, None, lambda g, a=False: (X.abs() if a else X).T @ g, dt == B, N, "dgate")


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_logits_gradient_joins_the_weights(shape):
    """router_backward with the weights' gradient, an addend and a gradient of the logits: dL/dlogits is their sum."""
    N, H, E, K, dt = shape
    say(f"[router grad_logits] {shape}")
    x, w, _, _ = _inputs(*shape, seed=1)
    g = torch.Generator().manual_seed(N)
    gw, gl = torch.randn(N, K, generator=g), torch.randn(N, E, generator=g) * 0.1
    add = torch.randn(N, H, generator=g).to(dt)
    xd, wd = x.to(dev()), w.to(dev())
    idx, _, logits, _, cnt, _ = ops.router_forward(xd, wd, K)
    lg = logits.cpu()
    G0 = OR.route_bwd(lg, idx.cpu(), gw)
    for addend in (None, add):
        dx, dw = ops.router_backward(xd, wd, logits, idx, gw.to(dev()), cnt, dx_add=None if addend is None else addend.to(dev()),
                                     grad_logits=gl.to(dev()))
        # the weights' term: probabilities and their quotients in fp32, a few tens of ulps of its largest terms
        mag = gl.double().abs() + G0.abs() + 2 * gw.double().abs().sum(1, keepdim=True) * torch.softmax(lg.double(), 1)
        room = 1.0 if addend is None else 2.0  # the router's part is rounded before the addend joins it
        W, X = w.double(), x.double()
        want = (G0 + gl.double()) @ W.T
        tol = ((3 * E + 300) * U * 4 + (2.0 ** -8 if dt == B else 0.0)) * (mag @ W.abs().T)
        tol = tol + room * (2.0 ** -8 if dt == B else U) * (want.abs() + tol) + 1e-30
        if addend is not None:
            want = want + addend.double()
            tol = tol + (2.0 ** -8 if dt == B else U) * (want.abs() + tol)
        off = ((dx.cpu().double() - want).abs() / tol).max()
        assert float(off) <= 1.0, f"dx: {float(off):.3f}"
        wantw = X.T @ (G0 + gl.double())
        tol = ((3 * E + 300) * U * 4 + (2.0 ** -8 if dt == B else 0.0) + N * U) * (X.abs().T @ mag)
        tol = tol + (2.0 ** -8 if dt == B else U) * (wantw.abs() + tol) + 1e-30
        off = ((dw.cpu().double() - wantw).abs() / tol).max()
        assert float(off) <= 1.0, f"dgate: {float(off):.3f}"
    # a gradient of zeros changes no bit
    a = ops.router_backward(xd, wd, logits, idx, gw.to(dev()), cnt)
    b = ops.router_backward(xd, wd, logits, idx, gw.to(dev()), cnt, grad_logits=torch.zeros(N, E, device=dev()))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("E", [8, 16, 64])
def test_norm_fused_router(E):
    """The same gradient behind the fused norm: against the router's own over the normalised rows, then the norm's backward."""
    N, H, K = 150, 512, 2
    say(f"[seq balance norm] E={E}")
    x, w, offs, mask = _inputs(N, H, E, K, B, seed=2)
    nw = 1.0 + 0.1 * torch.randn(H, generator=torch.Generator().manual_seed(3))
    xd, wd, nd = (t.to(dev()).requires_grad_(True) for t in (x, w, nw))
    xn, idx, _w, _a, _z, logits, cnt, _s = NormRouterCore.apply(xd, nd, 1e-5, wd, K, 0.0, 0.0, None, True)
    out = balance_loss(logits, idx, offs.to(dev()), mask.to(dev()), BC, ZC)
    dx, dn, dw = torch.autograd.grad(out[0] + out[1], (xd, nd, wd))
    d = ops.balance_loss_backward(logits.detach(), out[2], out[3], K, offs.to(dev()), mask.to(dev()), None, None, BC, ZC)
    G = d.double().cpu()
    W, XN = w.double(), xn.detach().double().cpu()
    want = XN.T @ G
    tol = (2.0 ** -8 + N * U) * (XN.abs().T @ G.abs())
    assert bool(((dw.double().cpu() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30).all())
    # the norm's backward of u = G W^T in float64; every rounding of u, dx is 2^-8 of a term at most
    X, N64 = x.double(), nw.double()
    r = torch.rsqrt((X * X).mean(1, keepdim=True) + 1e-5)
    xh = X * r
    u, room = G @ W.T, 2 * 2.0 ** -8 * (G.abs() @ W.abs().T)
    gx = u * N64
    ref = r * (gx - xh * (gx * xh).mean(1, keepdim=True))
    rr = room * N64.abs()
    tol = r * (rr + xh.abs() * (rr * xh.abs()).mean(1, keepdim=True)) * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs() + 1e-30
    off = ((dx.double().cpu() - ref).abs() / tol).max()
    assert float(off) <= 1.0, f"dx {float(off):.3f}"
    refn, tn = (u * xh).sum(0), (room * xh.abs()).sum(0) + N * U * (u * xh).abs().sum(0) + 1e-30
    off = ((dn.double().cpu() - refn).abs() / (tn * (1 + 2.0 ** -8))).max()
    assert float(off) <= 1.0, f"dnorm {float(off):.3f}"


def test_router_module():
    """The rows of a padded batch are its sequences; the mask leaves padding out of the balance and z losses, not of the
    routing; without the new arguments nothing changes."""
    say("[seq balance module]")
    torch.manual_seed(0)
    Bn, S, H, E, K = 4, 50, 256, 8, 2
    r = MoERouter(H, E, K, dtype=B, aux_loss_coef=0.01, z_loss_coef=ZC, seq_balance_coef=BC).to(dev())
    plain = MoERouter(H, E, K, dtype=B, aux_loss_coef=0.01, z_loss_coef=ZC).to(dev())
    plain.load_state_dict(r.state_dict())
    x = torch.randn(Bn, S, H, device=dev()).bfloat16()
    mask = torch.arange(S, device=dev()) < torch.tensor([[50], [1], [0], [33]], device=dev())
    a, b = r(x, token_mask=mask), plain(x)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert plain.last_seq_balance_loss is None and torch.equal(r.last_aux_loss, plain.last_aux_loss)
    ref = OB.balance(r._last_logits.cpu(), a[0].cpu(), torch.arange(0, 201, 50), mask.reshape(-1).cpu(), BC, ZC)
    assert torch.equal(r.last_seq_counts.cpu(), ref["counts"]) and torch.equal(r.last_seq_tokens.cpu(), ref["tokens"])
    assert abs(float(r.last_seq_balance_loss.detach()) - float(ref["balance"])) <= 200 * U * float(ref["balance"])
    assert abs(float(r.last_z_loss.detach()) - float(ref["z"])) <= 200 * U * float(ref["z"])
    assert not r._last_logits.requires_grad
    z_all = plain.last_z_loss
    r(x)  # no mask: the kernel's z-loss over every token
    assert torch.equal(r.last_z_loss, z_all) and int(r.last_seq_tokens[-2]) == Bn * S
    r(x.reshape(-1, H), seq_offsets=torch.tensor([0, 10, 200], device=dev()))
    assert r.last_seq_counts.shape == (2, E) and r.last_seq_tokens.tolist() == [10, 190, 200, 2]
    r.seq_balance_coef = 0.0
    r(x)
    assert r.last_seq_balance_loss is None


@pytest.mark.parametrize("E,dt", [(8, B), (64, B), (8, F)], ids=["E8-bf16", "E64-bf16", "E8-f32"])
def test_layer_and_block(E, dt):
    """Through the layer (tokens linked to the expert path) and the block (norm fused): the loss's gradient alone equals the
    whole backward's minus the backward without it, to the tokens' roundings."""
    say(f"[seq balance layer] E={E} {dt}")
    torch.manual_seed(1)
    H, Fd, K, Bn, S = 256, 128, 2, 3, 40
    x = torch.randn(Bn, S, H, device=dev()).to(dt).requires_grad_(True)
    mask = torch.rand(Bn, S, device=dev()) < 0.7
    gout = torch.randn(Bn, S, H, device=dev()).to(dt)
    for make in (lambda: DistributedMoELayer(H, Fd, E, K, build_topology(), dtype=dt, layout="routed", seq_balance_coef=20.0),
                 lambda: ToyMoEBlock(H, Fd, E, K, build_topology(), dtype=dt, layout="routed", seq_balance_coef=20.0)):
        m = make().to(dev())
        router = m.router if hasattr(m, "router") else m.moe.router
        out = m(x, token_mask=mask)
        both = torch.autograd.grad([out, router.last_seq_balance_loss], [x, router.gate_w], [gout, None])
        out2 = m(x, token_mask=mask)
        assert torch.equal(out, out2)
        alone = torch.autograd.grad(router.last_seq_balance_loss, [x, router.gate_w])
        out3 = m(x)
        rest = torch.autograd.grad(out3, [x, router.gate_w], gout)
        for a, b, c in zip(both, alone, rest):
            assert float(b.double().abs().max()) > 0
            eps = 2.0 ** -8 if dt == B else 64 * U
            # each gradient is rounded once or twice on its way (dL/dlogits, the output, a sum of two)
            off = (a.double() - b.double() - c.double()).norm() / (b.double().norm() + c.double().norm())
            assert float(off) <= 4 * eps, float(off)


def test_step_graph_replays_match_eager():
    """Routing with the balance loss, forward and backward, captured and replayed (as test_graph_gpu.py's steps: on one side
    stream, eager work between the replays)."""
    say("[seq balance graph]")
    from test_graph_gpu import _replays_match_eager

    x, w, offs, mask = _inputs(500, 512, 16, 4, B, seed=5)
    xd, wd = (t.to(dev()).requires_grad_(True) for t in (x, w))
    od, md = offs.to(dev()), mask.to(dev())
    gw = torch.randn(500, 4, device=dev()).bfloat16()
    one = torch.ones((), device=dev())

    def step():
        idx, wt, _aux, _z, logits, _cnt, _st = RouterCore.apply(xd, wd, 4, 0.0, 0.0, None, diff_logits=True)
        bal, z, counts, tokens, _ = balance_loss(logits, idx, od, md, BC, ZC)
        dx, dw = torch.autograd.grad((wt, bal, z), (xd, wd), grad_outputs=(gw, one, one))
        return idx, bal, z, counts, tokens, dx, dw

    _replays_match_eager(step, ("idx", "balance", "z", "counts", "tokens", "dx", "dgate"))
