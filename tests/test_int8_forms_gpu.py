"""Every form of the int8 products, shown to have run, at sizes just inside the rule that chooses it: whole rows and columns of
64 x 64 around each corner against the exact sums, with rows of no segment behind and experts without rows between."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import _lib, ops
from oracle import int8 as OI

pytestmark = pytest.mark.gpu

# name of the kernel, K, N, rows of each expert (None: one group of so many rows)
FORMS = [
    ("k_i8_small", 272, 520, [8, 0, 7, 1]),
    ("k_i8_small", 4096, 4096, 64),                   # one group, little to do
    ("k_i8_small", 144, 264, [1] + [0] * 200 + [1]),  # blocks for the experts with rows alone
    ("k_i8_small", 400, 264, [9, 3, 0, 21] * 20),     # many experts, little to do
    ("k_i8_tile192", 1040, 1032, [9, 3, 0, 21, 64, 65] * 12),
    ("k_i8_tile192", 1040, 1032, [9, 3, 0, 21, 64, 1, 65, 2] * 9),
    ("k_i8_tile192", 2048, 768, [2, 0, 200, 1] + [2] * 60),
    ("k_i8_tile64", 2048, 1016, [9, 3, 0, 21, 64, 1, 65, 2] * 9),
    ("k_i8_tile64", 2064, 776, [2, 0, 200, 1] + [3] * 124),
    ("k_i8_tile192", 1040, 4104, [20, 0, 193, 65, 1, 128, 10, 40]),
    ("k_i8_tile192", 2048, 4104, [300, 0, 383, 192, 129, 64, 500, 200]),
    ("k_i8_tile192_deep", 1024, 1032, [400, 0, 500, 64]),   # fewer tiles than CUs
    ("k_i8_tile192_turn", 1024, 1032, [400, 0, 129, 64]),
    ("k_i8_tile192_turn", 4096, 4104, [130, 70, 0, 50, 64, 60, 193, 100]),
    ("k_i8_tile192_turn", 4112, 8200, [130, 70, 0, 50, 64, 60, 192, 100]),
    ("k_i8_tile256", 272, 8200, [513 + 255, 700, 0, 900]),
    ("k_i8_tile256", 1024, 14344, 1025),
    ("k_i8_join", 14336, 520, 130),
    ("k_i8_join", 8192 + 16, 1032, [40, 0, 200, 100]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("form,K,N,counts", FORMS, ids=lambda v: str(v)[:20])
def test_product(form, K, N, counts, dtype):
    say(f"[int8 form] {form} K={K} N={N} {str(counts)[:40]} {dtype}")
    grouped = not isinstance(counts, int)
    counts = counts if grouped else [counts]
    E = len(counts)
    g = torch.Generator(device=dev()).manual_seed(K + N)
    used = sum(counts)
    R = used + (5 if grouped else 0)
    q = torch.randint(-127, 128, (R, K), device=dev(), generator=g, dtype=torch.int8)
    s = torch.rand(R, device=dev(), generator=g) + 0.5
    wq = torch.randint(-127, 128, (E, N, K), device=dev(), generator=g, dtype=torch.int8)
    ws = torch.rand(E, N, device=dev(), generator=g) * 1e-3 + 1e-4
    offs = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    _lib.prof_enable(True)
    y = ops.matmul_int8(q, s, wq if grouped else wq[0], ws if grouped else ws[0], offsets=offs.to(dev()) if grouped else None,
                        out_dtype=dtype)
    ran = set(_lib.prof_summary())
    _lib.prof_enable(False)
    assert form in ran, ran
    step = OI.BF16 if dtype == torch.bfloat16 else 0.0
    for e in range(E):
        lo, hi = int(offs[e]), int(offs[e + 1])
        if lo == hi or (E > 16 and e % 7 and counts[e] < 100):
            continue
        for cols in (slice(0, 128), slice(max(0, N // 2 - 64), N // 2 + 64), slice(max(0, N - 128), N)):
            want = OI.matmul(q[lo:hi], s[lo:hi], wq[e, cols], ws[e, cols])
            # the sum to fp32 and two products, then the type's rounding
            off = ((y[lo:hi, cols].double() - want).abs() / (want.abs() * (3.01 * OI.F32 + step) + 1e-45)).max()
            assert float(off) <= 1.0, f"expert {e} columns {cols}: {float(off):.3f} of the bound"


GATE_UP = [
    ("k_i8_small_gu", 144, 80, [8, 0, 7, 1]),
    ("k_i8_small_gu", 272, 144, [9, 3, 0, 21] * 20),
    ("k_i8_tile192_gu", 1040, 1040, [9, 3, 0, 21, 64, 1] * 12),
    ("k_i8_tile64_gu", 2048, 1008, [9, 3, 0, 21, 64, 1] * 12),
    ("k_i8_tile192_gu", 528, 3088, [20, 0, 193, 65, 1, 128, 10, 40]),
    ("k_i8_small_gu", 528, 1040, [300, 0, 65, 64]),
    ("k_i8_tile192_deep_gu", 528, 1040, [300, 0, 565, 64]),
    ("k_i8_tile192_turn_gu", 528, 2064, [300, 0, 365, 64]),
    ("k_i8_tile192_turn_gu", 4096, 4112, [130, 70, 0, 50, 64, 60, 192, 100]),
    ("k_i8_tile256_gu", 272, 4112, [513 + 255, 700, 0, 900]),
]


@pytest.mark.parametrize("form,H,F,counts", GATE_UP, ids=lambda v: str(v)[:20])
def test_experts(form, H, F, counts):
    say(f"[int8 experts form] {form} H={H} F={F} {str(counts)[:40]}")
    E, g = len(counts), torch.Generator(device=dev()).manual_seed(H + F)
    wq, ws = [], []
    for r, c in ((F, H), (F, H), (H, F)):
        a, b = ops.quant_rows_int8(torch.randn(E, r, c, device=dev(), generator=g) * c ** -0.5)
        wq.append(a)
        ws.append(b)
    offs = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    T = 97  # rows read any token, some never, some often
    q, s = ops.quant_rows_int8(torch.randn(T, H, device=dev(), generator=g))
    slot = torch.randint(0, 3 * T, (sum(counts),), device=dev(), generator=g, dtype=torch.int32)
    _lib.prof_enable(True)
    y = ops.swiglu_forward_int8(q, s, wq, ws, offs.to(dev()), row_slot=slot, top_k=3)
    ran = set(_lib.prof_summary())
    _lib.prof_enable(False)
    assert form in ran, ran
    token = (slot // 3).long()
    want, tol = OI.swiglu_fwd(q[token], s[token], wq, ws, offs.tolist())
    off = ((y.double() - want).abs() / tol).max()
    assert bool(torch.isfinite(y).all()) and float(off) <= 1.0, f"{float(off):.3f} of the bound"
