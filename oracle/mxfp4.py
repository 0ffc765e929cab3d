"""CPU restatement of the experts held in 4 bits (MXFP4) -- TEST INFRASTRUCTURE ONLY.

The reference has no 4-bit path (moe-engine's experts run in the model dtype: pkg/distributed/moe_layer.py L:166-198,
L:326-337); the contract is stated here:

* ``quant`` -- every 32 consecutive elements of a row share 2^e, e the smallest integer with absmax <= 6 * 2^e, clamped to
  [-124, 125], stored as the byte e + 127; elements x * 2^-e rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (ties to
  the one with an even code), at most 6, sign in bit 3; the even column in the low half of a byte.  A block with an
  infinity or a NaN has the byte 255.
* ``dequant`` -- the values, in float64; NaN in blocks of byte 255.
* ``swiglu_fwd`` / ``swiglu_bwd`` -- the experts on dequantized weights in float64, nothing rounded between, with a bound
  on what fp32 sums and the roundings to bf16 of act (forward) and dg, du (backward) may change (a rounding to bf16 is off by
  at most 2^-8 of the value, a sum of n terms in fp32 by n 2^-24 of the sum of their magnitudes).

Pinning (``tests/test_oracle_mxfp4.py``): ``quant`` by a brute-force search over exponents and values, ``dequant`` by its
table, ``swiglu_bwd`` by autograd of the forward's formula.
"""

from __future__ import annotations

from typing import Sequence, Tuple

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BF16, F32 = 2.0 ** -8, 2.0 ** -24


def quant(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    v = x.double().reshape(*x.shape[:-1], -1, 32)
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    m, p = torch.frexp(torch.where(bad, 1.0, amax))  # 6 = 0.75 * 2^3
    e = torch.where(m <= 0.75, p - 3, p - 2)
    e = torch.where(amax > 0, e, torch.full_like(e, -124)).clamp(-124, 125)
    a = torch.where(bad.unsqueeze(-1), 0.0, v.abs()) * torch.exp2(-e.double()).unsqueeze(-1)
    d = (a.clamp(max=6.0).unsqueeze(-1) - VALUES).abs()
    near = d == d.amin(-1, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.int().argmax(-1), near.int().argmax(-1))
    code = (code + 8 * (torch.signbit(v) & ~bad.unsqueeze(-1)).long()).to(torch.uint8)
    code = code.reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), torch.where(bad, 255, e + 127).to(torch.uint8)


def dequant(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    code = torch.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1).long()
    v = torch.cat([VALUES, -VALUES]).to(q.device)[code]
    s = torch.where(scale == 255, float("nan"), torch.exp2(scale.double() - 127))
    return v * s.repeat_interleave(32, -1)


def _sum(n: int, magnitudes: torch.Tensor) -> torch.Tensor:
    """Error of an fp32 sum of n products (any order, the products exact) with this sum of magnitudes."""
    return (n + 1) * F32 * magnitudes


def swiglu_fwd(x: torch.Tensor, w: Sequence[torch.Tensor], offsets: Sequence[int]):
    """(hgu [R, 2F], y [R, H]) in float64 for rows x [R, H] and dequantized weights (gate, up [E, F, H], down [E, H, F]),
    and how far the bf16 outputs may be off: (hgu_tol, y_tol).  Rows past offsets[E] are zero."""
    wg, wu, wd = w
    R, H = x.shape
    F = wg.shape[1]
    hgu, y = (torch.zeros(R, n, dtype=torch.float64, device=x.device) for n in (2 * F, H))
    ht, yt = torch.zeros_like(hgu), torch.zeros_like(y)
    for e in range(len(offsets) - 1):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        if s.start >= s.stop:
            continue
        xe = x[s].double()
        g, u = xe @ wg[e].T, xe @ wu[e].T
        dg, du = _sum(H, xe.abs() @ wg[e].abs().T), _sum(H, xe.abs() @ wu[e].abs().T)
        sig = torch.sigmoid(g)
        act = g * sig * u
        # |silu'| <= 1.1; the hardware's exp2, reciprocal and products: a few ulps, taken as 2^-20
        da = 1.1 * dg * (u.abs() + du) + (g * sig).abs() * du + 2.0 ** -20 * act.abs()
        da = da + BF16 * (act.abs() + da)
        hgu[s], ht[s] = torch.cat([g, u], 1), torch.cat([dg, du], 1)
        y[s] = act @ wd[e].T
        yt[s] = da @ wd[e].abs().T + _sum(F, (act.abs() + da) @ wd[e].abs().T)
    tiny = 2.0 ** -133  # half the smallest subnormal of bf16
    return hgu, y, ht + BF16 * (hgu.abs() + ht) + tiny, yt + BF16 * (y.abs() + yt) + tiny


def swiglu_bwd(dy: torch.Tensor, hgu: torch.Tensor, w: Sequence[torch.Tensor], offsets: Sequence[int]):
    """dxp [R, H] in float64 and how far the bf16 output may be off."""
    wg, wu, wd = w
    R, H = dy.shape
    F = wg.shape[1]
    dx = torch.zeros(R, H, dtype=torch.float64, device=dy.device)
    tol = torch.zeros_like(dx)
    for e in range(len(offsets) - 1):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        if s.start >= s.stop:
            continue
        d, g, u = dy[s].double(), hgu[s, :F].double(), hgu[s, F:].double()
        da = d @ wd[e]
        ta = _sum(H, d.abs() @ wd[e].abs())
        sig = torch.sigmoid(g)
        kg, ku = u * sig * (1 + g * (1 - sig)), g * sig
        # the factors in fp32: a few ulps of their terms, taken as 2^-19
        dg, du = da * kg, da * ku
        tg = ta * kg.abs() + 2.0 ** -19 * (da.abs() + ta) * (u * sig).abs() * (1 + g.abs())
        tu = ta * ku.abs() + 2.0 ** -19 * (da.abs() + ta) * ku.abs()
        tg, tu = tg + BF16 * (dg.abs() + tg), tu + BF16 * (du.abs() + tu)
        dx[s] = dg @ wg[e] + du @ wu[e]
        t = tg @ wg[e].abs() + tu @ wu[e].abs()
        tol[s] = t + _sum(2 * F, (dg.abs() + tg) @ wg[e].abs() + (du.abs() + tu) @ wu[e].abs())
    return dx, tol + BF16 * (dx.abs() + tol) + 2.0 ** -133
