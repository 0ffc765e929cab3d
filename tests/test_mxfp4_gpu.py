"""Experts held in 4 bits (MXFP4) on the GPU against oracle/mxfp4.py: the quantization bit-exact, the products within the
bounds that the oracle derives element by element from the roundings (fp32 sums, bf16 act / dg / du, bf16 outputs)."""

from __future__ import annotations

import threading

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import _lib, ops
from oracle import mxfp4 as OX

pytestmark = pytest.mark.gpu


def _same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=777.0), torch.nan_to_num(b, nan=777.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (65, 160), (300, 4096), (33, 14336), (2, 5, 64), (64,)], ids=str)
def test_quant_dequant_bit_exact(shape, dtype):
    say(f"[mxfp4 quant] {shape} {dtype}")
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g)
    x = (x * torch.exp2(torch.randint(-130, 127, shape[:-1] + (1,), generator=g).float())).to(dtype)
    f = x.view(-1)
    f[:10] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0]).to(dtype)  # ties
    f[10:32] = 0.0
    if f.numel() >= 96:
        f[40] = float("inf")
        f[70] = float("nan")
    if f.numel() >= 320:
        f[96:128] = 0.0                                     # a zero block
        f[128:160] = 0.0
        f[129] = torch.finfo(dtype).max                     # saturates at 6 * 2^125
        f[160:192] = torch.finfo(dtype).tiny / 64           # subnormals
        f[192:224] = 3.0 * 2.0 ** -5                        # exactly 6 * 2^e
    q, s = ops.quant_mxfp4(x.to(dev()))
    rq, rs = OX.quant(x)
    assert torch.equal(s.cpu(), rs), "scale bytes"
    live = (rs != 255).repeat_interleave(16, -1)
    assert torch.equal(q.cpu()[live], rq[live]), "4-bit pairs"
    for out in (torch.bfloat16, torch.float32):
        v = ops.dequant_mxfp4(q, s, out)
        assert v.dtype == out and v.shape == x.shape
        assert _same(v.cpu().double(), OX.dequant(rq, rs)), "values"


def test_quant_of_a_view_and_empty():
    x = torch.randn(64, 96, device=dev()).bfloat16()
    a, b = ops.quant_mxfp4(x.T[:, :64]), ops.quant_mxfp4(x.T[:, :64].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q, s = ops.quant_mxfp4(x[:0])
    assert q.shape == (0, 48) and s.shape == (0, 3) and ops.dequant_mxfp4(q, s).shape == (0, 96)


def _experts(E, F, H, seed):
    g = torch.Generator(device=dev()).manual_seed(seed)
    q, s, w = [], [], []
    for r, c in ((F, H), (F, H), (H, F)):
        t = torch.randn(E, r, c, device=dev(), generator=g) * c ** -0.5
        a, b = ops.quant_mxfp4(t)
        q.append(a)
        s.append(b)
        w.append(OX.dequant(a, b))
    return q, s, w


def _offsets(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)


def _inside(got, want, tol, what):
    off = ((got.double() - want).abs() / tol).max() if got.numel() else torch.tensor(0.0)
    assert bool(torch.isfinite(got).all()) and float(off) <= 1.0, f"{what}: {float(off):.3f} of the bound"


CASES = [
    (32, 32, [1]),                           # the smallest
    (32, 64, [0, 1, 0, 2]),                  # experts without rows
    (96, 160, [5, 17, 1]),                   # a partial 128-column chunk in both products
    (128, 128, [16, 32, 33, 64, 65, 1]),     # at the row passes' edges
    (160, 96, [3] * 130),                    # more than 128 experts
    (32, 32, [70, 5, 300]),                  # one block a row, many rows
    (96, 64, [100, 0, 257, 64]),             # rows of an odd number of blocks
    (288, 416, [500, 130]),                  # reductions that leave 32 of 128 columns
    (192, 224, [260, 0, 129]),               # ... 64 and 96
    (544, 1056, [127, 0, 129, 40]),          # odd blocks of a row
    (2048, 768, [9, 3, 0, 70]),
    (1024, 4096, [300, 0, 513, 1]),
    (4096, 14336, [1, 1]),                   # one decoded token
    (4096, 14336, [30, 140]),
]


@pytest.mark.parametrize("H,F,counts", CASES, ids=lambda v: str(v)[:24])
def test_forward(H, F, counts):
    say(f"[mxfp4 experts] H={H} F={F} counts={counts[:8]}")
    q, s, w = _experts(len(counts), F, H, H + F)
    offs = _offsets(counts)
    R = int(offs[-1]) + 3  # rows past the last segment
    x = torch.randn(R, H, device=dev(), generator=torch.Generator(device=dev()).manual_seed(R)).bfloat16()
    used = int(offs[-1])
    x[used:] = float("nan")
    hgu, y = ops.swiglu_forward_mxfp4(x, q, s, offs.to(dev()))
    rh, ry, th, ty = OX.swiglu_fwd(x[:used], w, offs.tolist())
    _inside(hgu[:used], rh, th, "hgu")
    _inside(y[:used], ry, ty, "y")
    none, y2 = ops.swiglu_forward_mxfp4(x, q, s, offs.to(dev()), keep_preact=False)
    assert none is None and torch.equal(y2[:used], y[:used])


@pytest.mark.parametrize("H,F,counts", CASES, ids=lambda v: str(v)[:24])
def test_backward(H, F, counts):
    say(f"[mxfp4 experts backward] H={H} F={F} counts={counts[:8]}")
    q, s, w = _experts(len(counts), F, H, H + F + 1)
    offs = _offsets(counts)
    used = int(offs[-1])
    g = torch.Generator(device=dev()).manual_seed(used)
    dy = torch.randn(used + 2, H, device=dev(), generator=g).bfloat16()
    hgu = torch.randn(used + 2, 2 * F, device=dev(), generator=g).bfloat16()
    dy[used:], hgu[used:] = float("nan"), float("nan")
    dx = ops.swiglu_backward_mxfp4(dy, hgu, q, s, offs.to(dev()))
    rx, tx = OX.swiglu_bwd(dy[:used], hgu[:used], w, offs.tolist())
    _inside(dx[:used], rx, tx, "dxp")


@pytest.mark.parametrize("H,F,counts", [
    (160, 8224, [1500, 0, 700]),             # tiles of 128 rows, odd numbers of blocks
    (4096, 14336, [1100, 1003]),
    (128, 16384, [1000, 0, 1303]),           # of 256 rows
], ids=lambda v: str(v)[:24])
def test_forward_of_many_rows(H, F, counts):
    test_forward(H, F, counts)


@pytest.mark.parametrize("H,F,counts", [
    (160, 2080, [3000, 0, 1201]),            # tiles of 128 rows; reductions and columns of odd numbers of blocks
    (96, 544, [64, 70, 58] * 44),            # ... of many experts
    (8224, 2016, [4133, 101]),               # of 256 rows for dxp
], ids=lambda v: str(v)[:24])
def test_backward_of_many_rows(H, F, counts):
    test_backward(H, F, counts)


def test_rows_past_the_last_segment_are_left_alone():
    """Through the C ABI, whose caller owns the outputs."""
    H, F, counts = 128, 96, [3, 0, 20]
    q, s, _ = _experts(3, F, H, 5)
    offs = _offsets(counts).to(dev())
    R = 30
    x = torch.randn(R, H, device=dev()).bfloat16()
    y = torch.full((R, H), 7.0, device=dev()).bfloat16()
    hgu = torch.full((R, 2 * F), 9.0, device=dev()).bfloat16()
    lib = _lib.load()
    n = lib.moe_swiglu_fwd_mxfp4_workspace(R, H, F, 3)
    ws = _lib.workspace(n, dev())
    p = [t.data_ptr() for pair in zip(q, s) for t in pair]
    _lib.check(lib.moe_swiglu_fwd_mxfp4(x.data_ptr(), *p, offs.data_ptr(), R, H, F, 3, hgu.data_ptr(), y.data_ptr(),
                                        ws.data_ptr(), n, _lib.stream_of(dev())), "moe_swiglu_fwd_mxfp4")
    assert bool((y[23:] == 7).all()) and bool((hgu[23:] == 9).all()) and not bool((y[:23] == 7).all(-1).any())
    dx = torch.full((R, H), 5.0, device=dev()).bfloat16()
    n = lib.moe_swiglu_bwd_mxfp4_workspace(R, H, F, 3)
    ws = _lib.workspace(n, dev())
    _lib.check(lib.moe_swiglu_bwd_mxfp4(y.data_ptr(), hgu.data_ptr(), *p, offs.data_ptr(), R, H, F, 3, dx.data_ptr(),
                                        ws.data_ptr(), n, _lib.stream_of(dev())), "moe_swiglu_bwd_mxfp4")
    assert bool((dx[23:] == 5).all()) and not bool((dx[:23] == 5).all(-1).any())


@pytest.mark.parametrize("H,F,counts", [(96, 160, [5, 17, 1]), (544, 1056, [127, 2, 129, 40]), (1024, 512, [300, 300, 1])],
                         ids=lambda v: str(v)[:24])
def test_a_row_or_a_weight_block_that_is_nan_stays_its_own(H, F, counts):
    say(f"[mxfp4 nan] H={H} F={F}")
    q, s, _ = _experts(len(counts), F, H, 11)
    offs = _offsets(counts)
    R = int(offs[-1])
    x = torch.randn(R, H, device=dev()).bfloat16()
    _, good = ops.swiglu_forward_mxfp4(x, q, s, offs.to(dev()), keep_preact=False)
    bad = x.clone()
    bad[R // 2, H - 1] = float("nan")
    bad[0, 0] = float("inf")
    _, y = ops.swiglu_forward_mxfp4(bad, q, s, offs.to(dev()), keep_preact=False)
    rows = [r for r in range(R) if r not in (0, R // 2)]
    assert torch.equal(y[rows], good[rows]) and bool(y[R // 2].isnan().all())
    s2 = [t.clone() for t in s]
    s2[2][1, 7, -1] = 255  # one block of the second expert's down projection
    _, y = ops.swiglu_forward_mxfp4(x, q, s2, offs.to(dev()), keep_preact=False)
    lo, hi = int(offs[1]), int(offs[2])
    assert bool(y[lo:hi, 7].isnan().all())
    y[lo:hi, 7] = good[lo:hi, 7]
    assert torch.equal(y, good)


def test_a_rows_bits_do_not_depend_on_its_neighbours():
    H, F = 544, 1056
    q, s, _ = _experts(2, F, H, 13)
    x = torch.randn(40, H, device=dev()).bfloat16()
    _, y = ops.swiglu_forward_mxfp4(x, q, s, _offsets([0, 40]).to(dev()), keep_preact=False)
    for n in (1, 16, 17, 33):
        _, z = ops.swiglu_forward_mxfp4(x[:n], q, s, _offsets([0, n]).to(dev()), keep_preact=False)
        assert torch.equal(z, y[:n]), n


def test_graph_replays_other_streams_and_threads():
    say("[mxfp4 graph]")
    H, F, counts = 512, 768, [1, 0, 9, 40]
    q, s, _ = _experts(4, F, H, 17)
    offs = _offsets(counts).to(dev())
    R = sum(counts)
    x = torch.randn(R, H, device=dev()).bfloat16()
    side = torch.cuda.Stream()

    def step(t):
        hgu, y = ops.swiglu_forward_mxfp4(t, q, s, offs)
        return y, ops.swiglu_backward_mxfp4(y, hgu, q, s, offs)

    want = [t.clone() for t in step(x)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
        buf = x.clone()
        step(buf)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(buf)
    for i in range(4):
        buf.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(buf)))
    fails = []

    def work(k):
        try:
            for _ in range(10):
                if not all(torch.equal(a, b) for a, b in zip(step(x), want)):
                    fails.append(k)
        except Exception as e:  # raised again by the test's own thread
            fails.append(e)

    ts = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not fails, fails


@pytest.mark.parametrize("rows", [3, 1200])
def test_weights_of_more_than_2_gb(rows):
    """Offsets past 32 bits: the last expert's weights lie behind 2^31 bytes of each matrix."""
    say(f"[mxfp4 large] rows={rows}")
    E, H, F = 76, 4096, 14336
    g = torch.Generator(device=dev()).manual_seed(rows)
    q, s = [], []
    for r, c in ((F, H), (F, H), (H, F)):
        q.append(torch.randint(0, 256, (E, r, c // 2), dtype=torch.uint8, device=dev(), generator=g))
        s.append(torch.randint(117, 121, (E, r, c // 32), dtype=torch.uint8, device=dev(), generator=g))
    assert q[0][-1].data_ptr() - q[0].data_ptr() > 2 ** 31
    offs = _offsets([0] * (E - 1) + [rows])
    x, dy = (torch.randn(rows, H, device=dev(), generator=g).bfloat16() for _ in range(2))
    hgu, y = ops.swiglu_forward_mxfp4(x, q, s, offs.to(dev()))
    dx = ops.swiglu_backward_mxfp4(dy, hgu, q, s, offs.to(dev()))
    w = [OX.dequant(a[-1:], b[-1:]) for a, b in zip(q, s)]
    rh, ry, th, ty = OX.swiglu_fwd(x, w, [0, rows])
    _inside(hgu, rh, th, "hgu")
    _inside(y, ry, ty, "y")
    rx, tx = OX.swiglu_bwd(dy, hgu, w, [0, rows])
    _inside(dx, rx, tx, "dxp")


def test_two_graphs_of_split_products():
    """Forms whose last tiles are split over the reduction: two graphs, each with its own workspaces, replayed in turn with
    eager calls between."""
    say("[mxfp4 two graphs]")
    H, F, counts = 1024, 1056, [300, 213, 0, 500]
    q, s, _ = _experts(4, F, H, 23)
    offs = _offsets(counts).to(dev())
    x = torch.randn(2, sum(counts), H, device=dev()).bfloat16()

    def step(t):
        hgu, y = ops.swiglu_forward_mxfp4(t, q, s, offs)
        return hgu, y, ops.swiglu_backward_mxfp4(y, hgu, q, s, offs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        buf = [x[0].clone(), x[1].clone()]
        step(buf[0])
    side.synchronize()
    graphs, outs = [], []
    for b in buf:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step(b))
        graphs.append(g)
    for i in range(3):
        for k in (1, 0):
            buf[k].copy_(x[k] * (i + 1))
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], step(buf[k]))), (i, k)


def test_refusals():
    H, F = 64, 96
    q, s, _ = _experts(2, F, H, 19)
    offs = _offsets([1, 1]).to(dev())
    x = torch.randn(2, H, device=dev()).bfloat16()
    f = ops.swiglu_forward_mxfp4
    with pytest.raises(TypeError):
        f(x.float(), q, s, offs)
    with pytest.raises(TypeError):
        f(x, [t.int() for t in q], s, offs)
    with pytest.raises(ValueError):
        f(x[:, :32].contiguous(), q, s, offs)
    with pytest.raises(ValueError):
        f(x, q, s, offs.long())
    with pytest.raises(ValueError):
        f(x, q, s, offs[:2])
    with pytest.raises(ValueError):
        f(x, [q[0], q[1], q[2][:, :, :16].contiguous()], s, offs)
    with pytest.raises(ValueError):
        f(x, q, [s[0][:, :, :1].contiguous(), s[1], s[2]], offs)
    with pytest.raises(TypeError):
        f(x, [q[0].transpose(0, 1), q[1], q[2]], s, offs)
    with pytest.raises(RuntimeError):
        f(x, q, s, offs.cpu())
    with pytest.raises(ValueError):
        ops.swiglu_backward_mxfp4(x, x, q, s, offs)
    with pytest.raises(ValueError):
        ops.quant_mxfp4(x[:, :48])
    with pytest.raises(TypeError):
        ops.quant_mxfp4(x.half())
    with pytest.raises(ValueError):
        ops.dequant_mxfp4(q[0], s[0][:, :, :1])
    hgu, y = f(x[:0], q, s, _offsets([0, 0]).to(dev()))
    assert hgu.shape == (0, 2 * F) and y.shape == (0, H)


def test_scale_bytes_at_the_ranges_ends():
    """Bytes that ``quant_mxfp4`` never writes: 0 stands for 2^-127, with values down to 2^-128 (subnormal in bf16 and fp32)."""
    q = (torch.arange(16) | (15 - torch.arange(16)) << 4).to(torch.uint8)  # every value, twice
    q, s = q.expand(6, 16).contiguous(), torch.tensor([[0], [1], [2], [3], [252], [255]], dtype=torch.uint8)
    for dt in (torch.bfloat16, torch.float32):
        assert _same(ops.dequant_mxfp4(q.to(dev()), s.to(dev()), dt).cpu().double(), OX.dequant(q, s))


@pytest.mark.parametrize("H,F,rows", [(64, 64, 3), (1568, 96, 40), (256, 256, 700), (160, 8224, 1500), (128, 16384, 1100)],
                         ids=str)
@pytest.mark.parametrize("byte", [0, 1, 2, 252])
def test_products_of_scale_bytes_at_the_ranges_ends(H, F, rows, byte):
    """Weights of one such byte against rows that bring the product back into range: a subnormal operand of a matrix
    instruction counts in full."""
    say(f"[mxfp4 scale byte] {byte} H={H} F={F} rows={rows}")
    g = torch.Generator(device=dev()).manual_seed(byte + H)
    q = [torch.randint(0, 256, (1, r, c // 2), dtype=torch.uint8, device=dev(), generator=g)
         for r, c in ((F, H), (F, H), (H, F))]
    r = 2.0 ** (115 - byte if byte < 3 else -122)  # rows x weights: some 2^-12 (2^3)
    x = (torch.randn(rows, H, device=dev(), generator=g) * r).bfloat16()
    offs = torch.tensor([0, rows], dtype=torch.int32, device=dev())

    def scales(gate, up, down):
        return [torch.full((*t.shape[:2], t.shape[2] // 16), b, dtype=torch.uint8, device=dev())
                for t, b in zip(q, (gate, up, down))]

    for gate, up in ((byte, 127), (127, byte)):  # (only the half of the matrix with that byte is looked at)
        s = scales(gate, up, 127 if byte < 3 else 100)
        t = torch.where(torch.arange(H, device=dev()) < 32, x, 0).bfloat16()  # one block a row: sums stay finite
        hgu, _ = ops.swiglu_forward_mxfp4(t, q, s, offs)
        w = [OX.dequant(a, b) for a, b in zip(q, s)]
        rh, _, th, _ = OX.swiglu_fwd(t, w, [0, rows])
        half = slice(0, F) if gate == byte else slice(F, 2 * F)
        _inside(hgu[:, half], rh[:, half], th[:, half], "hgu")
        assert float(rh[:, half].abs().median()) > 0
    s = scales(125, 125, byte)
    hgu = torch.randn(rows, 2 * F, device=dev(), generator=g).bfloat16()
    dx = ops.swiglu_backward_mxfp4(x, hgu, q, s, offs)
    rx, tx = OX.swiglu_bwd(x, hgu, [OX.dequant(a, b) for a, b in zip(q, s)], [0, rows])
    _inside(dx, rx, tx, "dxp")
