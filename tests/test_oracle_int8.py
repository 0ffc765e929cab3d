"""oracle/int8.py and the norm with a residual against rational arithmetic, integers and autograd (CPU)."""

from __future__ import annotations

from fractions import Fraction

import pytest
import torch

from oracle import int8 as OI
from oracle import norm as ON

pytestmark = pytest.mark.cpu


def _nearest_even(f: Fraction) -> int:
    n = f.numerator // f.denominator
    rest = f - n
    if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and n % 2):
        n += 1
    return n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_quant_by_rationals(dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 48, generator=g) * torch.exp2(torch.randint(-30, 30, (40, 1), generator=g).float())
    x = x.to(dtype)
    x[0] = 0
    x[1, :4] = torch.tensor([1.0, 0.5, -0.5, 2.0 ** -8]).to(dtype)
    x[1, 4:] = 0.25
    x[2] = 2.0 ** -110  # below the smallest a
    x[3, 0] = torch.finfo(dtype).max
    x[4, 5] = torch.finfo(dtype).tiny
    x[5] = (torch.arange(48) * 2 + 1).to(dtype)  # 127 is among them: odd halves of a = 127 * 2^k are ties
    x[5, 0], x[5, 1] = 127.0 * 2, 127.0
    q, s = OI.quant(x)
    for r in range(x.shape[0]):
        a = max(max(abs(Fraction(float(v))) for v in x[r]), Fraction(2) ** -100)
        assert Fraction(float(s[r])) == Fraction(float(torch.tensor(float(a), dtype=torch.float64) / 127.0))
        assert q[r].tolist() == [_nearest_even(127 * Fraction(float(v)) / a) for v in x[r]]


def test_quant_of_rows_that_are_not_finite():
    x = torch.ones(3, 16)
    x[0, 3], x[2, 0] = float("nan"), float("-inf")
    q, s = OI.quant(x)
    assert torch.isnan(s).tolist() == [True, False, True]
    assert (q[0] == 0).all() and (q[2] == 0).all() and (q[1] == 127).all()


def test_matmul_by_integers_and_experts_by_values():
    g = torch.Generator().manual_seed(5)
    q = torch.randint(-127, 128, (9, 32), generator=g, dtype=torch.int8)
    s = torch.rand(9, generator=g).double() * 0.1
    wq = [torch.randint(-127, 128, (2,) + sh, generator=g, dtype=torch.int8) for sh in ((16, 32), (16, 32), (32, 16))]
    ws = [torch.rand(t.shape[:2], generator=g).double() * 1e-3 for t in wq]
    y = OI.matmul(q, s, wq[0][0], ws[0][0])
    want = (q.long() @ wq[0][0].long().T).double() * s[:, None] * ws[0][0]
    assert torch.equal(y, want)
    y, tol = OI.swiglu_fwd(q, s, wq, ws, [0, 4, 8])
    assert (y[8] == 0).all() and (tol[8] == 0).all()
    for e, (lo, hi) in enumerate([(0, 4), (4, 8)]):
        x = q[lo:hi].double() * s[lo:hi, None]
        w = [t[e].double() * c[e][:, None] for t, c in zip(wq, ws)]
        act = torch.nn.functional.silu(x @ w[0].T) * (x @ w[1].T)
        plain = act @ w[2].T
        # rounded twice: to bf16, and to whole numbers of the row's scale
        slack = act.abs() * OI.BF16 + act.abs().amax(-1, keepdim=True) * (1 + OI.BF16) / 254
        assert ((y[lo:hi] - plain).abs() <= slack @ w[2].abs().T).all()
        # the bound stays within a step or two of the bf16 rounding
        assert (tol[lo:hi] <= y[lo:hi].abs() * 2 * OI.BF16 + (slack @ w[2].abs().T)).all()


def test_e4m3_values():
    table = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    v = torch.cat([table, (table[1:] + table[:-1]) / 2, torch.rand(1000).double() * 448])
    d = (v.unsqueeze(-1) - table).abs()
    near = d == d.amin(-1, keepdim=True)
    code = torch.where(near & (torch.arange(127) % 2 == 0), 1, 0)
    pick = torch.where(code.any(-1), code.argmax(-1), near.int().argmax(-1))
    assert torch.equal(OI.e4m3(v), table[pick]) and torch.equal(OI.e4m3(-v), -table[pick])


@pytest.mark.parametrize("grads", ["both", "xn", "h"])
def test_norm_residual_by_autograd(grads):
    g = torch.Generator().manual_seed(7)
    x, r = torch.randn(5, 24, generator=g).double(), torch.randn(5, 24, generator=g).double()
    w = torch.randn(24, generator=g).double()
    dxn, dh = torch.randn(5, 24, generator=g).double(), torch.randn(5, 24, generator=g).double()
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    h = leaves[0] + leaves[1]
    xn = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + 1e-5) * leaves[2]
    y, hh, rstd = ON.rmsnorm_residual_fwd(x, r, w)
    assert torch.allclose(y, xn.detach(), rtol=1e-12, atol=1e-12) and torch.equal(hh, h.detach())
    loss = (0 if grads == "h" else (xn * dxn).sum()) + (0 if grads == "xn" else (h * dh).sum())
    loss.backward()
    d, dw = ON.rmsnorm_residual_bwd(hh, w, None if grads == "h" else dxn, None if grads == "xn" else dh)
    for leaf in leaves[:2]:
        assert torch.allclose(leaf.grad, d, rtol=1e-11, atol=1e-12)
    assert torch.allclose(dw, torch.zeros_like(w) if leaves[2].grad is None else leaves[2].grad, rtol=1e-11, atol=1e-12)
