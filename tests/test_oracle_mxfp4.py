"""oracle/mxfp4.py against brute force and autograd, and the argument checks of the 4-bit entry points (CPU only: no call
here launches a kernel)."""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp4 as OX

from moe_mi355 import _lib, ops

pytestmark = pytest.mark.cpu


def test_quant_brute_force():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 32, generator=g, dtype=torch.float64).float() * torch.logspace(-37, 37, 40).unsqueeze(1)
    x[3] = 0.0
    x[4, :10] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0])
    x[4, 10:] = 0.0
    q, s = OX.quant(x)
    v = OX.dequant(q, s)
    grid = [m * t for m in (1, -1) for t in OX.VALUES.tolist()]
    for r in range(40):
        amax = float(x[r].abs().max())
        e = next(e for e in range(-124, 126) if amax <= 6.0 * 2.0 ** e or e == 125)
        assert int(s[r, 0]) == e + 127
        for c in range(32):
            t = float(x[r, c]) / 2.0 ** e
            best = min(abs(t - w) for w in grid)
            assert abs(t - float(v[r, c]) / 2.0 ** e) == best
    # ties to the even code
    assert (v[4, :10] / 1.0).tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0, -4.0]


def test_quant_ends_of_the_range():
    big = torch.finfo(torch.float32).max
    x = torch.zeros(5, 32)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = big, 2.0 ** -149, float("inf"), float("nan")
    q, s = OX.quant(x)
    v = OX.dequant(q, s)
    assert s[:, 0].tolist() == [252, 3, 255, 255, 3]
    assert float(v[0, 0]) == 6 * 2.0 ** 125 and bool((v[1] == 0).all()) and bool(v[2:4].isnan().all())
    assert torch.equal(v[0].bfloat16().double(), v[0])


def test_backward_against_autograd_and_differences():
    g = torch.Generator().manual_seed(1)
    R, H, F, E = 5, 32, 64, 2
    w = [torch.randn(E, *s, generator=g, dtype=torch.float64) * 0.3 for s in ((F, H), (F, H), (H, F))]
    x = torch.randn(R, H, generator=g, dtype=torch.float64)
    dy = torch.randn(R, H, generator=g, dtype=torch.float64)
    offs = [0, 3, 5]

    def f(t):
        out = []
        for e in range(E):
            xe = t[offs[e]:offs[e + 1]]
            out.append((torch.nn.functional.silu(xe @ w[0][e].T) * (xe @ w[1][e].T)) @ w[2][e].T)
        return (torch.cat(out) * dy).sum()

    xr = x.clone().requires_grad_(True)
    auto, = torch.autograd.grad(f(xr), xr)
    hgu, y, _, _ = OX.swiglu_fwd(x, w, offs)
    assert abs(float((y * dy).sum() - f(x))) < 1e-12
    dx, _ = OX.swiglu_bwd(dy, hgu, w, offs)
    assert float((dx - auto).abs().max()) < 1e-12
    for r, c in ((0, 0), (2, 31), (4, 7)):
        h = torch.zeros_like(x)
        h[r, c] = 1e-5
        assert abs(float(f(x + h) - f(x - h)) / 2e-5 - float(dx[r, c])) < 1e-7


def test_c_abi_refusals():
    lib = _lib.load()
    assert lib.moe_quant_mxfp4(None, 1, 4, 48, None, None, None) == -1 and "cols % 32" in _lib.last_error()
    assert lib.moe_quant_mxfp4(None, 7, 4, 64, None, None, None) == -1
    assert lib.moe_quant_mxfp4(None, 1, 4, 64, None, None, None) == -1 and "null" in _lib.last_error()
    assert lib.moe_quant_mxfp4(None, 1, 0, 64, None, None, None) == 0
    assert lib.moe_dequant_mxfp4(None, None, -1, 64, None, 1, None) == -1
    P = [None] * 8
    for R, H, F, E in ((-1, 64, 64, 4), (4, 48, 64, 4), (4, 64, 40, 4), (4, 64, 64, 1025), (4, 0, 64, 4)):
        assert lib.moe_swiglu_fwd_mxfp4(*P, R, H, F, E, None, None, None, 0, None) == -1
        assert "bad shape" in _lib.last_error()
        assert lib.moe_swiglu_bwd_mxfp4(*P, None, R, H, F, E, None, None, 0, None) == -1
    assert lib.moe_swiglu_fwd_mxfp4(*P, 4, 64, 64, 4, None, None, None, 0, None) == -1 and "null" in _lib.last_error()
    fake = 4096  # an aligned address that no call below reads: the workspace is refused first
    assert lib.moe_swiglu_fwd_mxfp4(*[fake] * 8, 4, 64, 64, 4, None, fake, fake, 16, None) == -2
    assert lib.moe_swiglu_fwd_mxfp4(*[fake] * 8, 4, 64, 64, 4, fake + 2, fake, fake, 1 << 20, None) == -1
    assert lib.moe_swiglu_bwd_mxfp4(*[fake] * 9, 4, 64, 64, 4, fake, fake, 16, None) == -2
    assert lib.moe_swiglu_fwd_mxfp4_workspace(0, 64, 64, 4) == 0


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        ops.quant_mxfp4(torch.zeros(4, 64))
    z = torch.zeros(1, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.swiglu_forward_mxfp4(torch.zeros(2, 64, dtype=torch.bfloat16), (z, z, z), (z, z, z), torch.zeros(2))
