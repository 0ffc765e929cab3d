"""CPU restatement of rows and weights held in int8 -- TEST INFRASTRUCTURE ONLY.

The reference has no integer path (moe-engine's experts run in the model dtype: pkg/distributed/moe_layer.py L:166-198,
L:326-337); the contract is stated here:

* ``quant`` -- with a = max(absmax of the row, 2^-100): scale = a / 127, each element the whole number nearest to 127 x / a,
  ties to even.  (For 24-bit values the quotient in float64 is never rounded onto a tie: two different quotients of such
  values by a border differ by more than 2^-34 of it.)  A row with an infinity or a NaN has the scale NaN and elements 0.
* ``matmul`` -- sx[m] sw[n] sum_k xq[m, k] wq[n, k] in float64 (the sum exact).
* ``swiglu_fwd`` -- the experts on int8 rows and weights with act rounded to bf16 and quantized by row, and a bound on what
  fp32 may change: an act next to a border of bf16 or of int8 may fall on its other side.

Pinning (``tests/test_oracle_int8.py``): ``quant`` by rational arithmetic, ``matmul`` by integers, ``swiglu_fwd`` by the
float64 layer on dequantized weights.
"""

from __future__ import annotations

from typing import Sequence, Tuple

import torch

TINY = 2.0 ** -100
BF16, F32 = 2.0 ** -8, 2.0 ** -24
E4M3_MAX = 448.0


def quant(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(whole numbers int8, scales float64) of rows [..., cols]."""
    v = x.double()
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad.unsqueeze(-1), 0.0, v)
    a = v.abs().amax(-1).clamp(min=TINY)
    q = torch.round(127.0 * v / a.unsqueeze(-1)).to(torch.int8)
    return q, torch.where(bad, float("nan"), a / 127.0)


def matmul(q: torch.Tensor, s: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor) -> torch.Tensor:
    return (q.double() @ wq.double().T) * s.double().unsqueeze(-1) * ws.double()


# g, u: the sum to fp32 and two products (3 roundings); silu: e^-g off by (|g| + 2) 2^-23 at most (its argument's rounding and
# the function's own), the sum, the reciprocal and two products 5 more
def _act_error(g: torch.Tensor, act: torch.Tensor) -> torch.Tensor:
    return act.abs() * F32 * (6.0 + 2.0 * (4.0 * g.abs() + 2.0) + 5.0)


def swiglu_fwd(q: torch.Tensor, s: torch.Tensor, wq: Sequence[torch.Tensor], ws: Sequence[torch.Tensor],
               offsets: Sequence[int]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y [R, H] float64, how far a bf16 y may be off) for rows q [R, H] grouped by expert; rows past offsets[E] are zero.

    |silu'(g)| <= 1.1 and silu(g) >= |g| e^-|g| / 2 for g < 0, so a relative error e of g moves silu by at most
    (1 + |g|) e of itself: the 4 |g| in the bound."""
    R, H = q.shape
    y = torch.zeros(R, H, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(y)
    for e in range(len(offsets) - 1):
        lo, hi = offsets[e], offsets[e + 1]
        if lo >= hi:
            continue
        g = matmul(q[lo:hi], s[lo:hi], wq[0][e], ws[0][e])
        u = matmul(q[lo:hi], s[lo:hi], wq[1][e], ws[1][e])
        act = g * torch.sigmoid(g) * u
        err = _act_error(g, act)
        low, high = (act - err).to(torch.bfloat16).double(), (act + err).to(torch.bfloat16).double()
        a = act.to(torch.bfloat16).double()
        aq, sa = quant(a)
        # the row's scale, and each element's whole number, over what act may have been rounded to
        m = a.abs().amax(-1)
        top = torch.maximum(low.abs(), high.abs()).amax(-1)
        bot = torch.minimum(low.abs(), high.abs()).amax(-1)
        dscale = torch.where(m > 0, (top - bot) / m.clamp(min=TINY), torch.zeros_like(m)).unsqueeze(-1)  # 0 almost always
        step = torch.where(low != high, (high - low).abs() / sa.unsqueeze(-1) + 1.0, 0.0)
        step = torch.where(dscale > 0, step + 1.0 + aq.double().abs() * dscale, step)
        down, sd = wq[2][e].double(), ws[2][e].double()
        y[lo:hi] = (aq.double() @ down.T) * sa.unsqueeze(-1) * sd
        slack = (step @ down.abs().T) * sa.unsqueeze(-1) * sd
        tol[lo:hi] = slack + (y[lo:hi].abs() + slack) * (BF16 + dscale + 8 * F32) + 2.0 ** -133
    return y, tol


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value in float64: three bits behind the leading one, exponents from -6, at most 448; ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
