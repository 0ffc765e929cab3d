"""Rows and weights in int8 on the GPU against oracle/int8.py: quantization bit-exact, products exact up to the scales'
roundings, experts within the bound that the oracle derives from what fp32 may round differently."""

from __future__ import annotations

import threading

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import _lib, ops
from oracle import int8 as OI

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(16,), (1, 16), (3, 48), (65, 512), (130, 528), (33, 2048), (9, 4112), (5, 14336), (3, 16384),
                                   (2, 16400), (2, 40000), (2, 5, 64), (9000, 32), (8300, 1024)], ids=str)
def test_quant_dequant_bit_exact(shape, dtype):
    say(f"[int8 quant] {shape} {dtype}")
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g)
    x = (x * torch.exp2(torch.randint(-60, 60, shape[:-1] + (1,), generator=g).float())).to(dtype)
    rows = x.view(-1, shape[-1])
    if rows.shape[0] >= 3:
        rows[0] = 0.0
        rows[1, : shape[-1] // 2] = rows[1].abs().max() / 2  # every one on the border between 63 and 64
        rows[2, -1] = torch.finfo(dtype).max
    if rows.shape[0] >= 9:
        rows[3, 5] = float("inf")
        rows[4, shape[-1] - 1] = float("nan")
        rows[5] = torch.finfo(dtype).tiny
        rows[6] = (torch.arange(shape[-1]) % 254 - 127).to(dtype) * 0.5
        rows[6, 0] = 127.0
        rows[7] *= 2.0 ** -126
    q, s = ops.quant_rows_int8(x.to(dev()))
    rq, rs = OI.quant(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == x.shape and s.shape == x.shape[:-1]
    assert torch.equal(q.cpu(), rq), f"{(q.cpu() != rq).sum()} of {rq.numel()} whole numbers differ"
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(rs.float(), nan=-1.0)), "scales"
    for out in (torch.bfloat16, torch.float32):
        v = ops.dequant_rows(q, s, out)
        want = (rq.float() * rs.float().unsqueeze(-1)).to(out)  # one fp32 product, then the rounding
        assert v.dtype == out and torch.equal(torch.nan_to_num(v.cpu(), nan=777.0), torch.nan_to_num(want, nan=777.0))


def test_every_border_of_every_bf16_row_maximum():
    # a row for each mantissa of its largest value, and in it every half step that bf16 or fp32 holds next to the border
    a = 1.0 + torch.arange(128, dtype=torch.float64) / 128
    n = torch.arange(127, dtype=torch.float64)
    border = ((2 * n + 1) / 254).unsqueeze(0) * a.unsqueeze(1)
    b = border.float()
    x = torch.cat([b, torch.nextafter(b, b * 0), torch.nextafter(b, b * 2), a.float().unsqueeze(1)], 1)
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 16))
    x = torch.cat([x, -x, x * 2.0 ** -90, x * 2.0 ** 100, x.bfloat16().float()])
    q, s = ops.quant_rows_int8(x.to(dev()))
    rq, rs = OI.quant(x)
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs.float())


def test_dequant_of_e4m3_bytes():
    x = torch.randn(70, 144, device=dev(), generator=_gen(1))
    x[3] = 0
    q, s = ops.quant_rows_fp8(x)
    for out in (torch.bfloat16, torch.float32):
        v = ops.dequant_rows(q, s, out)
        assert torch.equal(v, (q.view(torch.float8_e4m3fn).float() * s.unsqueeze(-1)).to(out))


def test_quant_of_a_view_and_of_nothing():
    x = torch.randn(64, 96, device=dev()).bfloat16()
    a, b = ops.quant_rows_int8(x.T[:, :48]), ops.quant_rows_int8(x.T[:, :48].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q, s = ops.quant_rows_int8(x[:0])
    assert q.shape == (0, 96) and s.shape == (0,) and ops.dequant_rows(q, s).shape == (0, 96)


def _rows(R, K, seed):
    """Whole numbers that no quantization is needed for, largest ones among them."""
    q = torch.randint(-127, 128, (R, K), device=dev(), generator=_gen(seed), dtype=torch.int8)
    s = torch.rand(R, device=dev(), generator=_gen(seed + 1)) * 0.02 + 1e-3
    if R > 1:
        q[1] = 127
    return q, s


def _weights(E, N, K, seed):
    q = torch.randint(-127, 128, (E, N, K), device=dev(), generator=_gen(seed), dtype=torch.int8)
    q[:, 0] = 127  # the largest sum there is, with the row of 127s
    return q, torch.rand(E, N, device=dev(), generator=_gen(seed + 1)) * 1e-3 + 1e-5


def _check_product(y, want, dtype, what):
    # the sum to fp32 and two products: 3 roundings; then the type's own
    tol = want.abs() * (3.01 * OI.F32 + (OI.BF16 if dtype == torch.bfloat16 else 0.0)) + 1e-45
    off = ((y.double() - want).abs() / tol).max() if y.numel() else torch.tensor(0.0)
    assert bool(torch.isfinite(y).all()) and float(off) <= 1.0, f"{what}: {float(off):.3f} of the bound"


PRODUCTS = [
    (1, 16, 8), (2, 32, 24), (16, 48, 16), (17, 4096, 4096), (33, 144, 40), (64, 128, 128), (65, 272, 264), (100, 2064, 1000),
    (127, 512, 256), (128, 640, 520), (130, 4096, 520), (257, 1024, 776), (500, 96, 2000), (1000, 14336, 1024), (1, 14336, 4096),
    (3, 131056, 16), (2049, 768, 1032), (40, 14336, 8),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("R,K,N", PRODUCTS, ids=str)
def test_product(R, K, N, dtype):
    say(f"[int8 product] R={R} K={K} N={N} {dtype}")
    q, s = _rows(R, K, R + K)
    wq, ws = _weights(1, N, K, N + K)
    y = ops.matmul_int8(q, s, wq[0], ws[0], out_dtype=dtype)
    assert y.shape == (R, N) and y.dtype == dtype
    _check_product(y, OI.matmul(q, s, wq[0], ws[0]), dtype, "y")


GROUPS = [
    (16, 8, [1]), (32, 24, [0, 3, 0, 17]), (128, 64, [16, 32, 33, 64, 65, 1]), (144, 72, [3] * 130), (96, 40, [70, 5, 300]),
    (2048, 768, [129, 0, 300, 1, 255, 256, 257, 64]), (272, 264, [128, 127, 520]), (4096, 264, [30, 140, 0, 9]),
    (512, 512, [1] * 1024), (640, 136, [2000, 1, 0, 33]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("K,N,counts", GROUPS, ids=lambda v: str(v)[:24])
def test_grouped_product(K, N, counts, dtype):
    say(f"[int8 groups] K={K} N={N} counts={counts[:8]} {dtype}")
    E = len(counts)
    offs = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    used = int(offs[-1])
    q, s = _rows(used + 3, K, K + N)
    s[used:] = float("nan")
    wq, ws = _weights(E, N, K, N)
    y = ops.matmul_int8(q, s, wq, ws, offsets=offs.to(dev()), out_dtype=dtype)
    assert y.shape == (used + 3, N)
    for e in range(E):
        lo, hi = int(offs[e]), int(offs[e + 1])
        if lo < hi and (E < 64 or e % 37 == 0):
            _check_product(y[lo:hi], OI.matmul(q[lo:hi], s[lo:hi], wq[e], ws[e]), dtype, f"expert {e}")


def _into(entry, y, *args):
    """A call of the C ABI on the current stream, y already there."""
    rc = getattr(_lib.load(), entry)(*args, _lib.stream_of(y.device))
    _lib.check(rc, entry)


def _product_into(q, s, wq, ws, offs, y):
    E = wq.shape[0] if wq.dim() == 3 else 1
    n = _lib.load().moe_matmul_int8_workspace(q.shape[0], q.shape[1], wq.shape[-2], E)
    w = _lib.workspace(n, dev())
    _into("moe_matmul_int8", y, q.data_ptr(), s.data_ptr(), wq.data_ptr(), ws.data_ptr(), _lib.ptr(offs), q.shape[0],
          q.shape[1], wq.shape[-2], E, y.data_ptr(), _lib.dtype_code(y.dtype), w.data_ptr(), n)


@pytest.mark.parametrize("counts", [[3, 0, 9], [200, 0, 90], [700, 0, 600]], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_rows_of_no_segment_are_left_as_they_were(counts, dtype):
    K, N = 144, 136
    offs = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=dev())
    used = sum(counts)
    q, s = _rows(used + 300, K, 1)
    wq, ws = _weights(3, N, K, 2)
    y = torch.full((used + 300, N), 7.5, device=dev(), dtype=dtype)
    _product_into(q, s, wq, ws, offs, y)
    assert (y[used:] == 7.5).all() and (y[:used] != 7.5).any(-1).all()


def test_a_rows_result_is_the_same_in_any_batch():
    K, N = 1040, 264
    q, s = _rows(900, K, 3)
    wq, ws = _weights(1, N, K, 4)
    full = ops.matmul_int8(q, s, wq[0], ws[0])
    for lo, hi in [(0, 1), (5, 21), (100, 164), (37, 300), (1, 900)]:
        assert torch.equal(ops.matmul_int8(q[lo:hi], s[lo:hi], wq[0], ws[0]), full[lo:hi])


def test_product_of_more_dims_and_of_views():
    q, s = _rows(24, 96, 5)
    wq, ws = _weights(1, 40, 96, 6)
    flat = ops.matmul_int8(q, s, wq[0], ws[0])
    assert torch.equal(ops.matmul_int8(q.view(2, 3, 4, 96), s.view(2, 3, 4), wq[0], ws[0]), flat.view(2, 3, 4, 40))
    assert torch.equal(ops.matmul_int8(q[0], s[0], wq[0], ws[0]), flat[0])
    wide = torch.cat([q, q], 1)
    assert torch.equal(ops.matmul_int8(wide[:, 96:], s, wq[0], ws[0]), flat)
    assert ops.matmul_int8(q[:0], s[:0], wq[0], ws[0]).shape == (0, 40)


# ---- the experts ----


def _experts(E, F, H, seed):
    out = [[], []]
    for i, (r, c) in enumerate(((F, H), (F, H), (H, F))):
        t = torch.randn(E, r, c, device=dev(), generator=_gen(seed + i)) * c ** -0.5
        a, b = ops.quant_rows_int8(t)
        out[0].append(a)
        out[1].append(b)
    return out


def _inside(got, want, tol, what):
    off = ((got.double() - want).abs() / tol).max() if got.numel() else torch.tensor(0.0)
    assert bool(torch.isfinite(got).all()) and float(off) <= 1.0, f"{what}: {float(off):.3f} of the bound"


CASES = [
    (16, 16, [1]),                           # the smallest
    (32, 48, [0, 1, 0, 2]),                  # experts without rows
    (96, 160, [5, 17, 1]),
    (128, 128, [16, 32, 33, 64, 65, 1]),     # at the row passes' edges
    (160, 96, [3] * 130),                    # more than 128 experts
    (32, 32, [70, 5, 300]),
    (272, 400, [500, 130]),                  # reductions that leave 16 of 128 columns
    (208, 240, [260, 0, 129]),
    (544, 1040, [127, 0, 129, 40]),
    (2048, 768, [9, 3, 0, 70]),
    (1024, 4096, [300, 0, 513, 1]),
    (4096, 14336, [1, 1]),                   # one decoded token
    (4096, 14336, [30, 140]),
    (512, 1024, [1200, 800]),
]


@pytest.mark.parametrize("H,F,counts", CASES, ids=lambda v: str(v)[:24])
def test_experts(H, F, counts):
    say(f"[int8 experts] H={H} F={F} counts={counts[:8]}")
    wq, ws = _experts(len(counts), F, H, H + F)
    offs = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    used = int(offs[-1])
    x = torch.randn(used + 3, H, device=dev(), generator=_gen(used)).bfloat16()  # rows past the last segment
    x[used:] = float("nan")
    q, s = ops.quant_rows_int8(x)
    y = ops.swiglu_forward_int8(q, s, wq, ws, offs.to(dev()))
    ry, ty = OI.swiglu_fwd(q[:used], s[:used], wq, ws, offs.tolist())
    assert y.shape == (used + 3, H) and y.dtype == torch.bfloat16
    _inside(y[:used], ry, ty, "y")


@pytest.mark.parametrize("T,K,E,H,F", [(1, 2, 8, 96, 64), (7, 3, 5, 144, 80), (64, 8, 128, 256, 96), (300, 2, 4, 272, 144),
                                       (1500, 4, 3 + 1, 128, 256)], ids=str)
def test_rows_read_through_the_plan(T, K, E, H, F):
    say(f"[int8 gather] T={T} K={K} E={E}")
    wq, ws = _experts(E, F, H, T)
    x = torch.randn(T, H, device=dev(), generator=_gen(T)).bfloat16()
    idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:K] for t in range(T)]).to(dev())
    p = ops.plan(idx, E, layout=ops.LAYOUT_ROUTED)
    q, s = ops.quant_rows_int8(x)
    y = ops.swiglu_forward_int8(q, s, wq, ws, p.offsets, row_slot=p.row_slot, top_k=K)
    token = (p.row_slot // K).long()
    assert torch.equal(y, ops.swiglu_forward_int8(q[token], s[token], wq, ws, p.offsets))
    ry, ty = OI.swiglu_fwd(q[token], s[token], wq, ws, p.offsets.tolist())
    _inside(y, ry, ty, "y")


def test_a_token_that_is_not_finite_spoils_its_own_rows_alone():
    E, F, H = 3, 64, 96
    wq, ws = _experts(E, F, H, 1)
    offs = torch.tensor([0, 40, 40, 100], dtype=torch.int32, device=dev())
    x = torch.randn(100, H, device=dev(), generator=_gen(2)).bfloat16()
    clean = ops.swiglu_forward_int8(*ops.quant_rows_int8(x), wq, ws, offs)
    x[17, 3], x[60, 0] = float("inf"), float("nan")
    y = ops.swiglu_forward_int8(*ops.quant_rows_int8(x), wq, ws, offs)
    bad = torch.zeros(100, dtype=torch.bool, device=dev())
    bad[17] = bad[60] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


def test_experts_leave_rows_of_no_segment_alone():
    E, F, H, R = 2, 64, 96, 500
    wq, ws = _experts(E, F, H, 1)
    for counts in ([5, 9], [300, 100]):
        offs = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device=dev())
        q, s = _rows(R, H, 3)
        y = torch.full((R, H), 7.5, device=dev(), dtype=torch.bfloat16)
        n = _lib.load().moe_swiglu_fwd_int8_workspace(R, H, F, E)
        w = _lib.workspace(n, dev())
        w.fill_(255)  # NaNs behind the last segment's rows
        _into("moe_swiglu_fwd_int8", y, q.data_ptr(), s.data_ptr(), R, None, 1, wq[0].data_ptr(), ws[0].data_ptr(),
              wq[1].data_ptr(), ws[1].data_ptr(), wq[2].data_ptr(), ws[2].data_ptr(), offs.data_ptr(), R, H, F, E, y.data_ptr(),
              w.data_ptr(), n)
        used = sum(counts)
        assert (y[used:] == 7.5).all()
        assert torch.equal(y[:used], ops.swiglu_forward_int8(q, s, wq, ws, offs)[:used])


# ---- streams, graphs, threads ----


@pytest.mark.parametrize("T,K,E,H,F", [(4, 2, 8, 256, 128), (900, 2, 4, 256, 384)], ids=["few", "many"])
def test_captured_and_replayed(T, K, E, H, F):
    wq, ws = _experts(E, F, H, 7)
    idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:K] for t in range(T)]).to(dev())
    p = ops.plan(idx, E, layout=ops.LAYOUT_ROUTED)
    x = torch.randn(T, H, device=dev(), generator=_gen(1)).bfloat16()

    def step():
        q, s = ops.quant_rows_int8(x)
        y = ops.swiglu_forward_int8(q, s, wq, ws, p.offsets, row_slot=p.row_slot, top_k=K)
        return y, ops.matmul_int8(q, s, wq[0][0], ws[0][0]), ops.dequant_rows(q, s)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                out = step()
            graphs.append((g, out))
        for i in range(4):
            x.copy_(torch.randn(T, H, device=dev(), generator=_gen(100 + i)).bfloat16())
            for g, _ in graphs:
                g.replay()
            stream.synchronize()
            want = step()
            stream.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {i}"
    torch.cuda.current_stream().wait_stream(stream)


def test_threads_on_one_stream_and_on_their_own():
    E, F, H = 4, 128, 256
    wq, ws = _experts(E, F, H, 7)
    jobs = []
    for i, R in enumerate((3, 60, 700, 1200)):
        c = R // E
        offs = torch.tensor([0, c, 2 * c, 3 * c, R], dtype=torch.int32, device=dev())
        q, s = ops.quant_rows_int8(torch.randn(R, H, device=dev(), generator=_gen(i)).bfloat16())
        jobs.append((q, s, offs, ops.swiglu_forward_int8(q, s, wq, ws, offs)))
    torch.cuda.synchronize()
    for own_stream in (False, True):
        bad = []

        def work(job):
            q, s, offs, want = job
            with torch.cuda.stream(torch.cuda.Stream() if own_stream else torch.cuda.current_stream()):
                for _ in range(20):
                    y = ops.swiglu_forward_int8(q, s, wq, ws, offs)
                torch.cuda.current_stream().synchronize()
            if not torch.equal(y, want):
                bad.append(q.shape)

        ts = [threading.Thread(target=work, args=(j,)) for j in jobs]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        assert not bad


# ---- refusals ----


def test_refusals():
    q, s = _rows(8, 96, 1)
    wq, ws = _weights(2, 40, 96, 2)
    offs = torch.tensor([0, 4, 8], dtype=torch.int32, device=dev())
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.quant_rows_int8(q)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.quant_rows_int8(torch.zeros(4, 40, device=dev()))
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        ops.dequant_rows(q, s, torch.float16)
    with pytest.raises(ValueError, match="scale must be"):
        ops.dequant_rows(q, s[:4])
    with pytest.raises(TypeError, match="int8"):
        ops.matmul_int8(q.float(), s, wq[0], ws[0])
    with pytest.raises(TypeError, match="weights are int8"):
        ops.matmul_int8(q, s, wq[0].float(), ws[0])
    with pytest.raises(ValueError, match=r"\[E, N, K\]"):
        ops.matmul_int8(q, s, wq[0], ws[0], offsets=offs)
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        ops.matmul_int8(q, s, wq, ws)
    with pytest.raises(ValueError, match="do not go with"):
        ops.matmul_int8(q[:, :80].contiguous(), s, wq[0], ws[0])
    with pytest.raises(ValueError, match="contiguous"):
        ops.matmul_int8(q, s, wq.transpose(1, 2).contiguous().transpose(1, 2)[0], ws[0])
    with pytest.raises(ValueError, match="offsets must be"):
        ops.matmul_int8(q, s, wq, ws, offsets=offs.long())
    with pytest.raises(ValueError, match="offsets must be"):
        ops.matmul_int8(q, s, wq, ws, offsets=offs[:2])
    with pytest.raises(ValueError, match="N %"):
        ops.matmul_int8(q, s, wq[0, :36], ws[0, :36])
    with pytest.raises(ValueError, match="misaligned"):
        ops.matmul_int8(torch.zeros(8 * 96 + 8, dtype=torch.int8, device=dev())[8:].view(8, 96), s, wq[0], ws[0])
    with pytest.raises(RuntimeError, match="AMD Instinct"):
        ops.matmul_int8(q.cpu(), s, wq[0], ws[0])
    eq, es = _experts(2, 64, 96, 3)
    with pytest.raises(ValueError, match="down must be"):
        ops.swiglu_forward_int8(q, s, (eq[0], eq[1], eq[0]), es, offs)
    with pytest.raises(ValueError, match="up scale must be"):
        ops.swiglu_forward_int8(q, s, eq, (es[0], es[2], es[2]), offs)
    with pytest.raises(ValueError, match="row_slot must be"):
        ops.swiglu_forward_int8(q, s, eq, es, offs, row_slot=torch.zeros(8, dtype=torch.int64, device=dev()), top_k=2)
    with pytest.raises(ValueError, match="row_slot must be"):
        ops.swiglu_forward_int8(q, s, eq, es, offs, row_slot=torch.zeros(8, dtype=torch.int32, device=dev()), top_k=0)
    assert ops.swiglu_forward_int8(q[:0], s[:0], eq, es, offs * 0).shape == (0, 96)


def _lowest(shape, seed):
    """Any int8 values, -128 (which quantization never writes) often among them."""
    q = torch.randint(-128, 128, shape, device=dev(), generator=_gen(seed), dtype=torch.int8)
    return torch.where(torch.rand(shape, device=dev(), generator=_gen(seed + 1)) < 0.25, -128, q.int()).to(torch.int8)


@pytest.mark.parametrize("R,K,N", [(1, 4096, 4096), (16, 48, 16), (64, 4096, 4096), (300, 2048, 1032), (1100, 1024, 1544),
                                   (64, 14336, 520), (3, 131056, 16), (70, 131056, 1024)], ids=str)
def test_product_of_the_lowest_values(R, K, N):
    """Weights and rows of -128: scales of 1, so the result is the sum, rounded to fp32 once.  Its largest, 128 * 128 * 131056, is
    below 2^31."""
    say(f"[int8 -128] R={R} K={K} N={N}")
    q, wq = _lowest((R, K), 1), _lowest((N, K), 2)
    q[0] = wq[0] = wq[N - 1] = -128
    y = ops.matmul_int8(q, torch.ones(R, device=dev()), wq, torch.ones(N, device=dev()), out_dtype=torch.float32)
    want = (q.double() @ wq.double().T).float()  # whole numbers below 2^53: exact
    assert torch.equal(y, want)


def test_experts_on_the_lowest_values():
    E, H, F, counts = 4, 272, 144, [3, 0, 70, 17]
    wq = [_lowest(sh, 3 + i) for i, sh in enumerate(((E, F, H), (E, F, H), (E, H, F)))]
    ws = [torch.rand(t.shape[:2], device=dev(), generator=_gen(9)) * 1e-3 + 1e-4 for t in wq]
    for t in wq:
        t[:, 1] = -128
    offs = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    q, s = _lowest((sum(counts), H), 20), torch.rand(sum(counts), device=dev(), generator=_gen(21)) * 0.02 + 1e-3
    y = ops.swiglu_forward_int8(q, s, wq, ws, offs.to(dev()))
    want, tol = OI.swiglu_fwd(q, s, wq, ws, offs.tolist())
    assert float(((y.double() - want).abs() / tol).max()) <= 1.0
