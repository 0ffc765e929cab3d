"""The norm with the residual's addition, its backward, and its outputs in 8 bits, against oracle/norm.py and oracle/int8.py."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import ops
from oracle import int8 as OI
from oracle import norm as ON

pytestmark = pytest.mark.gpu

EPS = 1e-5
BF16, F32 = OI.BF16, OI.F32
SHAPES = [(1, 8), (3, 16), (5, 512), (1030, 64), (7, 520), (33, 2048), (9, 2064), (300, 4096), (5, 8192), (1, 4096), (4100, 96)]
DTYPES = [torch.bfloat16, torch.float32]


def _gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def _case(N, H, dtype, wdtype=torch.float32, seed=0):
    def t(std=1.0, shape=(N, H), dt=dtype):
        return (torch.randn(shape, device=dev(), generator=_gen(seed + len(made))) * std).to(dt)
    made = []
    for std in (1.0, 2.0, 1.0, 1.0):
        made.append(t(std))
    w = (1.0 + 0.1 * torch.randn(H, device=dev(), generator=_gen(seed + 9))).to(wdtype)
    return (*made, w)


def _step(dtype):
    return BF16 if dtype == torch.bfloat16 else F32


def _rel_rstd(H):
    """Relative error of rstd in fp32: H squares summed in lanes of H / 64 (at most 128) terms and six levels, half of it after
    the root; the mean, the sum with eps and the root itself, 4 more."""
    return ((max(8, H / 64) * 2 + 8) / 2 + 4) * F32


def _off(got, want, tol):
    return float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("wdtype", DTYPES, ids=["wbf16", "wf32"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("N,H", SHAPES, ids=str)
def test_forward(N, H, dtype, wdtype):
    say(f"[norm residual] N={N} H={H} {dtype} {wdtype}")
    x, r, _, _, w = _case(N, H, dtype, wdtype)
    xn, h, rstd = ops.rmsnorm_residual_forward(x, r, w, EPS)
    want, rh, rr = ON.rmsnorm_residual_fwd(x, r, w, EPS)
    assert torch.equal(h, rh)
    assert _off(rstd, rr, rr * _rel_rstd(H)) <= 1
    assert _off(xn, want, want.abs() * (_rel_rstd(H) + 2 * F32 + _step(dtype)) + 1e-37) <= 1
    # the norm alone, of h
    xn2, rstd2 = ops.rmsnorm_forward(h, w, EPS)
    assert torch.equal(xn, xn2) and torch.equal(rstd, rstd2)


@pytest.mark.parametrize("grads", ["both", "xn", "h"])
@pytest.mark.parametrize("wdtype", DTYPES, ids=["wbf16", "wf32"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("N,H", SHAPES, ids=str)
def test_backward(N, H, dtype, wdtype, grads):
    say(f"[norm residual bwd] N={N} H={H} {dtype} {wdtype} {grads}")
    x, r, dxn, dh, w = _case(N, H, dtype, wdtype)
    dxn, dh = (None if grads == "h" else dxn), (None if grads == "xn" else dh)
    _, h, rstd = ops.rmsnorm_residual_forward(x, r, w, EPS)
    d, dw = ops.rmsnorm_residual_backward(h, w, rstd, dxn, dh)
    rd, rdw = ON.rmsnorm_residual_bwd(h, w, dxn, dh, EPS)
    assert d.dtype == dtype and dw.dtype == wdtype
    v, rr = h.double(), torch.rsqrt(h.double().pow(2).mean(-1, keepdim=True) + EPS)
    u = torch.zeros_like(v) if dxn is None else dxn.double()
    e = _rel_rstd(H)
    g, xhat = (u * w.double()).abs(), (v * rr).abs()
    # mean(g xhat): every term off by e and 3 roundings, its sum by as many as rstd's
    dot = (g * xhat).mean(-1, keepdim=True)
    slack = rr * (g * (e + 4 * F32) + xhat * dot * (2 * e + 2 * e + 8 * F32)) + (rd.abs() + rr * (g + xhat * dot)) * 3 * F32
    assert _off(d, rd, slack + rd.abs() * _step(dtype) + 1e-37) <= 1
    # dweight: sums of N terms, each off by e and two roundings.  The longest chain of additions that a term goes through: a
    # lane's rows (up to 512 elements a wave a row, 2048 of them at once: N / 2048 + 1, then 3 waves; past that a block a row,
    # 1024 of them: N / 1024 + 1), the blocks' partial sums (at most 1024 / 32 in a row, then 31 more), the last rounding: at
    # most N / 1024 + 66, and 2 for the term itself
    sdw = (u * v * rr).abs().sum(0) * (e + (N / 1024 + 68) * F32)
    assert _off(dw, rdw, sdw + rdw.abs() * _step(wdtype) + 1e-37) <= 1


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_backward_by_differences(dtype):
    N, H = 3, 48
    x, r, dxn, dh, w = _case(N, H, dtype, seed=40)
    _, h, rstd = ops.rmsnorm_residual_forward(x, r, w, EPS)
    d, dw = ops.rmsnorm_residual_backward(h, w, rstd, dxn, dh)

    def loss(hh, ww):
        return (ON.rmsnorm_fwd(hh, ww, EPS)[0] * dxn.double()).sum() + (hh.double() * dh.double()).sum()

    step = 1e-5
    for i, j in [(0, 0), (1, 17), (2, 47)]:
        up, down = h.double(), h.double()
        up[i, j] += step
        down[i, j] -= step
        want = (loss(up, w.double()) - loss(down, w.double())) / (2 * step)
        # second-order terms of the difference are below 1e-8; d is rounded to its type and off by fp32 sums
        assert abs(float(d[i, j]) - float(want)) <= abs(float(want)) * _step(dtype) + 1e-5
        wu, wd = w.double(), w.double()
        wu[j] += step
        wd[j] -= step
        want = (loss(h, wu) - loss(h, wd)) / (2 * step)
        assert abs(float(dw[j]) - float(want)) <= 1e-5 * (1 + abs(float(want)))


@pytest.mark.parametrize("keep", [False, True], ids=["", "keep"])
@pytest.mark.parametrize("residual", [False, True], ids=["", "residual"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("N,H", [s for s in SHAPES if s[1] % 16 == 0], ids=str)
def test_rows_in_8_bits(N, H, dtype, fmt, residual, keep):
    say(f"[norm quant] N={N} H={H} {dtype} {fmt} residual={residual} keep={keep}")
    x, r, _, _, w = _case(N, H, dtype, seed=20)
    if N >= 5:
        x[2], r[2] = 0, 0  # a row of zeros
    q, s, xn, h = ops.rmsnorm_quant(x, w, EPS, residual=r if residual else None, fmt=fmt, keep_norm=keep)
    if residual:
        want, rh, _ = ON.rmsnorm_residual_fwd(x, r, w, EPS)
        assert torch.equal(h, rh)
    else:
        want = ON.rmsnorm_fwd(x, w, EPS)[0]
        rh = x
        assert h is None
    if keep:  # the very rows of the norm alone
        assert torch.equal(xn, ops.rmsnorm_forward(rh, w, EPS)[0])
    else:
        assert xn is None
    e = _rel_rstd(H) + 2 * F32  # of every normalised value
    amax = want.abs().amax(-1)
    value = ops.dequant_rows(q, s, torch.float32)
    if fmt == "int8":
        assert q.dtype == torch.int8
        a = amax.clamp(min=OI.TINY)
        assert _off(s, a / 127, a / 127 * (e + F32) + 1e-45) <= 1
        # half a step of the scale, what the value and the scale are off by, and dequantization's rounding
        tol = (a / 127).unsqueeze(-1) * 0.5 * (1 + e + 2 * F32) + want.abs() * (2 * e + 4 * F32) + 1e-45
        assert _off(value, want, tol) <= 1
        exact = (torch.round(127 * want / a.unsqueeze(-1)) != q.double()).double().mean()
        assert float(exact) <= 4 * 127 * 2 * e + 1e-3  # only values next to a border fall on its other side
    else:
        assert q.dtype == torch.uint8
        a = torch.where(amax < 2.0 ** -118, torch.full_like(amax, OI.E4M3_MAX), amax)
        assert _off(s, a / OI.E4M3_MAX, a / OI.E4M3_MAX * (e + F32)) <= 1
        # half a step of e4m3 (2^-4 of the value, at least half of 2^-9), and as above
        sc = (a / OI.E4M3_MAX).unsqueeze(-1)
        tol = torch.maximum(want.abs() * 2.0 ** -4, sc * 2.0 ** -10) * (1 + 4 * e) + want.abs() * (2 * e + 4 * F32) + 1e-45
        assert _off(value, want, tol) <= 1


def test_quant_rows_of_the_norm_itself():
    """With fp32 rows the 8-bit output is the quantization of the norm's own output."""
    x, r, _, _, w = _case(70, 1040, torch.float32, seed=3)
    for fmt, quant in (("int8", ops.quant_rows_int8), ("e4m3", ops.quant_rows_fp8)):
        q, s, xn, _ = ops.rmsnorm_quant(x, w, EPS, residual=r, fmt=fmt, keep_norm=True)
        q2, s2 = quant(xn)
        assert torch.equal(q, q2) and torch.equal(s, s2)


def test_rows_that_are_not_finite():
    x, r, _, _, w = _case(9, 64, torch.bfloat16, seed=3)
    clean = ops.rmsnorm_quant(x, w, EPS, residual=r)
    x[4, 7] = float("nan")
    r[6, 1] = float("inf")
    q, s, _, h = ops.rmsnorm_quant(x, w, EPS, residual=r)
    ok = torch.ones(9, dtype=torch.bool, device=dev())
    ok[4] = ok[6] = False
    assert torch.isnan(s[~ok]).all() and (q[~ok] == 0).all()
    assert torch.equal(q[ok], clean[0][ok]) and torch.equal(s[ok], clean[1][ok])
    assert torch.isnan(h[4, 7]) and torch.isinf(h[6, 1])


def test_views_and_nothing():
    x, r, dxn, dh, w = _case(40, 64, torch.bfloat16, seed=5)
    xt, rt = x.T.contiguous().T, torch.cat([r, r], 1)[:, 64:]
    for a, b in zip(ops.rmsnorm_residual_forward(xt, rt, w, EPS), ops.rmsnorm_residual_forward(x, r, w, EPS)):
        assert torch.equal(a, b)
    xn, h, rstd = ops.rmsnorm_residual_forward(x[:0], r[:0], w, EPS)
    assert xn.shape == h.shape == (0, 64) and rstd.shape == (0,)
    d, dw = ops.rmsnorm_residual_backward(h, w, rstd, dxn[:0], dh[:0])
    assert d.shape == (0, 64) and (dw == 0).all()
    q, s, xn, h = ops.rmsnorm_quant(x[:0], w, EPS, residual=r[:0], keep_norm=True)
    assert q.shape == xn.shape == h.shape == (0, 64) and s.shape == (0,)


def test_captured_and_replayed():
    x, r, dxn, dh, w = _case(130, 512, torch.bfloat16, seed=6)

    def step():
        xn, h, rstd = ops.rmsnorm_residual_forward(x, r, w, EPS)
        d, dw = ops.rmsnorm_residual_backward(h, w, rstd, dxn, dh)
        q, s, xq, hq = ops.rmsnorm_quant(x, w, EPS, residual=r, keep_norm=True)
        return xn, h, d, dw, q, s, xq, hq

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = step()
        for i in range(3):
            x.copy_(torch.randn(130, 512, device=dev(), generator=_gen(60 + i)).bfloat16())
            g.replay()
            stream.synchronize()
            want = step()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {i}"
    torch.cuda.current_stream().wait_stream(stream)


def test_refusals():
    x, r, dxn, dh, w = _case(4, 64, torch.bfloat16, seed=7)
    with pytest.raises(TypeError, match="residual must have x's dtype"):
        ops.rmsnorm_residual_forward(x, r.float(), w, EPS)
    with pytest.raises(ValueError, match="residual must be"):
        ops.rmsnorm_residual_forward(x, r[:1], w, EPS)
    with pytest.raises(ValueError, match="weight"):
        ops.rmsnorm_residual_forward(x, r, w[:32], EPS)
    with pytest.raises(ValueError, match="8 <= H <= 8192"):
        ops.rmsnorm_residual_forward(torch.zeros(1, 8200, device=dev()), torch.zeros(1, 8200, device=dev()),
                                     torch.zeros(8200, device=dev()), EPS)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.rmsnorm_quant(x.half(), w, EPS)
    with pytest.raises(ValueError, match="H % 16"):
        ops.rmsnorm_quant(x[:, :24].contiguous(), w[:24], EPS)
    with pytest.raises(ValueError, match="fmt"):
        ops.rmsnorm_quant(x, w, EPS, fmt="fp8")
    xn, h, rstd = ops.rmsnorm_residual_forward(x, r, w, EPS)
    with pytest.raises(ValueError, match="needs a gradient"):
        ops.rmsnorm_residual_backward(h, w, rstd, None, None)
    with pytest.raises(TypeError, match="dh must have"):
        ops.rmsnorm_residual_backward(h, w, rstd, dxn, dh.float())
    with pytest.raises(ValueError, match="rstd must be"):
        ops.rmsnorm_residual_backward(h, w, rstd[:2], dxn, dh)
    with pytest.raises(RuntimeError, match="AMD Instinct"):
        ops.rmsnorm_quant(x.cpu(), w.cpu(), EPS)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("H", [64, 512, 2064, 8192])
def test_rows_in_8_bits_that_are_not_finite(H, dtype, fmt):
    """A row with an infinity or a NaN, before or after the residual's addition or made by the weight, has the scale NaN and
    elements 0, so that all of it reads back as NaNs; the others keep their bits."""
    x, r, _, _, w = _case(11, H, dtype, seed=3)
    x[1] = 0
    r[1] = 0
    clean = ops.rmsnorm_quant(x, w, EPS, residual=r, fmt=fmt, keep_norm=True)
    x[4, 7] = float("nan")
    r[6, 1] = float("inf")
    x[7, H - 1] = -float("inf")
    x[8, 0], r[8, 0] = float("inf"), -float("inf")
    x[9, :] = float("nan")
    q, s, xn, h = ops.rmsnorm_quant(x, w, EPS, residual=r, fmt=fmt, keep_norm=True)
    bad = torch.zeros(11, dtype=torch.bool, device=dev())
    bad[[4, 6, 7, 8, 9]] = True
    assert torch.isnan(s[bad]).all() and (q[bad] == 0).all()
    assert torch.isnan(ops.dequant_rows(q, s, torch.float32)[bad]).all()
    for a, b in zip((q, s, xn, h), clean):
        assert torch.equal(a[~bad], b[~bad])
    # the rows kept beside them are those of the norm alone
    assert torch.equal(torch.nan_to_num(xn.float(), nan=777.0), torch.nan_to_num(ops.rmsnorm_forward(h, w, EPS)[0].float(), nan=777.0))
    # finite rows whose normalised values are not
    wbad = w.clone()
    wbad[5] = float("inf")
    q, s, _, _ = ops.rmsnorm_quant(r[:4], wbad, EPS, fmt=fmt)
    assert torch.isnan(s).all() and (q == 0).all()  # (row 1: 0 times infinity)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("N,H", [(1, 8), (7, 64), (6, 520), (1030, 2048), (5, 8192)], ids=str)
def test_backward_of_the_sum_alone(N, H, dtype):
    """Without a gradient of the norm's output d is dh and dweight zero, whatever h holds (a padded row's values, say)."""
    x, r, _, dh, w = _case(N, H, dtype, seed=8)
    x[0, 0] = float("nan")
    r[N // 2, H - 1] = float("inf")
    r[N - 1, 3] = -float("inf")
    _, h, rstd = ops.rmsnorm_residual_forward(x, r, w, EPS)
    for wd in (w, w.bfloat16()):
        d, dw = ops.rmsnorm_residual_backward(h, wd, rstd, None, dh)
        assert torch.equal(d, dh) and d.data_ptr() != dh.data_ptr()
        assert dw.dtype == wd.dtype and (dw == 0).all()
