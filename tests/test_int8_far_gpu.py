"""int8 products whose rows, weights or experts lie farther than 31 or 32 bits reach, in each form of the kernels, against the exact
sums of some columns."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import ops
from oracle import int8 as OI

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def _bytes(*shape, seed):
    """Random int8 of more elements than one call of the generator takes."""
    out = torch.empty(shape, dtype=torch.int8, device=dev())
    flat, g = out.view(-1), _gen(seed)
    for at in range(0, flat.numel(), 1 << 30):
        flat[at: at + (1 << 30)].random_(-127, 128, generator=g)
    return out


def _check(y, q, s, wq, ws, what):
    # the sum to fp32 and two products: 3 roundings; then bf16's
    want = OI.matmul(q, s, wq, ws)
    off = ((y.double() - want).abs() / (want.abs() * (3.01 * OI.F32 + OI.BF16) + 1e-45)).max()
    assert bool(torch.isfinite(y).all()) and float(off) <= 1.0, f"{what}: {float(off):.3f} of the bound"


# rows of the product (an expert), K, N: N K is above 2^31, two experts are above 2^32
@pytest.mark.parametrize("rows,K,N", [(4, 131056, 20000), (40, 16384, 140000), (100, 16384, 140000), (1000, 16400, 140008)], ids=str)
def test_matrices_past_two_gigabytes(rows, K, N):
    say(f"[int8 far] {rows} rows, K={K} N={N}")
    wq = _bytes(2, N, K, seed=rows)
    ws = torch.rand(2, N, device=dev(), generator=_gen(1)) + 0.5
    q, s = _bytes(2 * rows, K, seed=2), torch.rand(2 * rows, device=dev(), generator=_gen(3)) + 0.5
    y = ops.matmul_int8(q, s, wq, ws, offsets=torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=dev()))
    one = ops.matmul_int8(q[rows:], s[rows:], wq[1], ws[1])
    cols = torch.cat([torch.arange(64), torch.randint(0, N, (64,), generator=torch.Generator().manual_seed(4)),
                      torch.arange(N - 64, N)]).to(dev())
    for e in range(2):
        r = slice(e * rows, (e + 1) * rows)
        _check(y[r][:, cols], q[r], s[r], wq[e][cols], ws[e][cols], f"expert {e}")
    assert torch.equal(one, y[rows:])


@pytest.mark.parametrize("R", [6, 60, 1500, 4000], ids=str)
def test_tokens_past_two_gigabytes(R):
    T, H, F, E = 1040000, 4096, 256, 2  # the last rows begin just below 2^32
    say(f"[int8 far tokens] R={R}")
    q, s = _bytes(T, H, seed=R), torch.rand(T, device=dev(), generator=_gen(1)) + 0.5
    wq, ws = [], []
    for i, (n, k) in enumerate([(F, H), (F, H), (H, F)]):
        a, b = ops.quant_rows_int8(torch.randn(E, n, k, device=dev(), generator=_gen(i)) * k ** -0.5)
        wq.append(a)
        ws.append(b)
    slot = torch.randint(0, 2 * T, (R,), device=dev(), generator=_gen(7)).to(torch.int32)
    slot[0], slot[R - 1] = 0, 2 * T - 1
    offs = torch.tensor([0, R // 3, R], dtype=torch.int32, device=dev())
    token = (slot // 2).long()
    y = ops.swiglu_forward_int8(q, s / 64, wq, ws, offs, row_slot=slot, top_k=2)
    assert torch.equal(y, ops.swiglu_forward_int8(q[token], s[token] / 64, wq, ws, offs))
    ry, ty = OI.swiglu_fwd(q[token], s[token] / 64, wq, ws, offs.tolist())
    off = ((y.double() - ry).abs() / ty).max()
    assert float(off) <= 1.0, f"{float(off):.3f} of the bound"
    with pytest.raises(ValueError, match="T H must be below"):
        ops.swiglu_forward_int8(torch.empty(1 << 20, H, dtype=torch.int8, device=dev()), torch.empty(1 << 20, device=dev()), wq, ws,
                                offs, row_slot=slot, top_k=2)


def test_long_rows_and_many_rows_in_8_bits():
    # more than 2^32 elements: rows of 4096, the last of them checked
    N, H = (1 << 20) + 9, 4096
    say("[int8 far rows]")
    x = torch.empty(N, H, dtype=torch.bfloat16, device=dev()).normal_(generator=_gen(5))
    w = torch.ones(H, device=dev())
    tail = slice(N - 64, N)
    q, s = ops.quant_rows_int8(x)
    tq, ts = ops.quant_rows_int8(x[tail])
    assert torch.equal(q[tail], tq) and torch.equal(s[tail], ts)
    assert torch.equal(ops.dequant_rows(q, s, torch.bfloat16)[tail], ops.dequant_rows(tq, ts, torch.bfloat16))
    q, s, xn, h = ops.rmsnorm_quant(x, w, 1e-5, residual=x, keep_norm=True)
    tq, ts, txn, th = ops.rmsnorm_quant(x[tail], w, 1e-5, residual=x[tail], keep_norm=True)
    assert torch.equal(q[tail], tq) and torch.equal(s[tail], ts) and torch.equal(xn[tail], txn) and torch.equal(h[tail], th)
    del q, xn
    xn, h, rstd = ops.rmsnorm_residual_forward(x, x, w, 1e-5)
    d, _ = ops.rmsnorm_residual_backward(h, w, rstd, xn, x)
    td, _ = ops.rmsnorm_residual_backward(h[tail], w, rstd[tail], xn[tail], x[tail])
    assert torch.equal(xn[tail], txn) and torch.equal(d[tail], td)
