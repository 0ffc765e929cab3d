"""The forms of the 4-bit experts' products, each shown to be the one that ran: through the C ABI, whose caller owns the
workspace, where the row tiles and the partial tiles of a split last round can be seen."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say
from test_mxfp4_gpu import _experts, _inside, _offsets

from moe_mi355 import _lib, ops
from oracle import mxfp4 as OX

pytestmark = pytest.mark.gpu

FILL = 0xA5


class _Product:
    """One call through the C ABI: its outputs, the row tiles that it ran and whether it wrote partial tiles."""

    def __init__(self, name, R, H, F, E, held):
        lib = _lib.load()
        self.n = getattr(lib, f"moe_swiglu_{name}_mxfp4_workspace")(R, H, F, E)
        self.ws = torch.full((self.n,), FILL, dtype=torch.uint8, device=dev())
        self.E, self.parts_at = E, lib.moe_swiglu_workspace(E) + (R * F * held + 255) // 256 * 256

    def tiles(self):
        return int(self.ws[: 4 * (self.E + 1)].view(torch.int32)[-1])

    def split(self):
        return bool((self.ws[self.parts_at:] != FILL).any())


def _forward(x, q, s, offs, F):
    R, H = x.shape
    E = offs.numel() - 1
    p = _Product("fwd", R, H, F, E, 2)
    hgu, y = x.new_empty((R, 2 * F)), torch.empty_like(x)
    w = [t.data_ptr() for pair in zip(q, s) for t in pair]
    _lib.check(_lib.load().moe_swiglu_fwd_mxfp4(x.data_ptr(), *w, offs.data_ptr(), R, H, F, E, hgu.data_ptr(), y.data_ptr(),
                                                p.ws.data_ptr(), p.n, _lib.stream_of(dev())), "moe_swiglu_fwd_mxfp4")
    return hgu, y, p


def _backward(dy, hgu, q, s, offs, F):
    R, H = dy.shape
    E = offs.numel() - 1
    p = _Product("bwd", R, H, F, E, 4)
    dx = torch.empty_like(dy)
    w = [t.data_ptr() for pair in zip(q, s) for t in pair]
    _lib.check(_lib.load().moe_swiglu_bwd_mxfp4(dy.data_ptr(), hgu.data_ptr(), *w, offs.data_ptr(), R, H, F, E, dx.data_ptr(),
                                                p.ws.data_ptr(), p.n, _lib.stream_of(dev())), "moe_swiglu_bwd_mxfp4")
    return dx, p


@pytest.fixture(scope="module")
def large():
    """Ten experts of 268 MB a matrix: the last one's weights lie behind 2^31 bytes of each."""
    E, H, F = 10, 16384, 32768
    g = torch.Generator(device=dev()).manual_seed(3)
    q, s = [], []
    for r, c in ((F, H), (F, H), (H, F)):
        q.append(torch.randint(0, 256, (E, r, c // 2), dtype=torch.uint8, device=dev(), generator=g))
        s.append(torch.randint(116, 120, (E, r, c // 32), dtype=torch.uint8, device=dev(), generator=g))
    assert q[0][-1].data_ptr() - q[0].data_ptr() > 2 ** 31
    yield E, H, F, q, s, [OX.dequant(a[-1:], b[-1:]) for a, b in zip(q, s)]


@pytest.mark.parametrize("rows,fwd,bwd", [(100, 0, 64), (200, 64, 64), (700, 64, 128), (1700, 128, 128), (5300, 256, 128),
                                          (10300, 256, 256)])
def test_weights_of_more_than_2_gb_in_every_form(large, rows, fwd, bwd):
    """``fwd`` and ``bwd``: the rows of the forward's and of dxp's tiles (0: the few-row form)."""
    say(f"[mxfp4 large forms] rows={rows}")
    E, H, F, q, s, w = large
    offs = _offsets([0] * (E - 1) + [rows]).to(dev())
    g = torch.Generator(device=dev()).manual_seed(rows)
    x, dy = (torch.randn(rows, H, device=dev(), generator=g).bfloat16() for _ in range(2))
    hgu, y, p = _forward(x, q, s, offs, F)
    if fwd:
        assert p.tiles() == -(-rows // fwd)
    else:
        assert bool((p.ws[:44] == FILL).all())  # no table of tiles
    dx, p = _backward(dy, hgu, q, s, offs, F)
    assert p.tiles() == -(-rows // bwd)
    # rows stand alone: the first and last, those at the tiles' edges, and some between
    pick = sorted({0, 63, 64, 127, 128, 255, 256, rows // 3, rows // 2, rows - 2, rows - 1} & set(range(rows)))
    n = [0, len(pick)]
    rh, ry, th, ty = OX.swiglu_fwd(x[pick], w, n)
    _inside(hgu[pick], rh, th, "hgu")
    _inside(y[pick], ry, ty, "y")
    rx, tx = OX.swiglu_bwd(dy[pick], hgu[pick], w, n)
    _inside(dx[pick], rx, tx, "dxp")


@pytest.mark.parametrize("H,F,counts,fwd,dxp,split", [
    (1024, 4096, [300, 0, 513, 1], 64, 64, (True, True)),          # the down projection and dxp split
    (4096, 4096, [700, 600], 64, 64, (False, True)),               # dact and dxp
    (160, 2080, [3000, 0, 1201], 64, 128, (True, True)),           # dxp of 128 rows, odd numbers of blocks
    (256, 8192, [1300, 1400], 128, 128, (True, True)),
    (128, 16384, [1000, 0, 1303], 256, 128, (True, True)),
    (8192, 2048, [4200], 64, 256, (True, True)),                   # dact of 128 rows, dxp of 256
], ids=lambda v: str(v)[:24])
def test_two_graphs_of_products_that_are_split(H, F, counts, fwd, dxp, split):
    """Products whose last tiles are split over the reduction: two graphs, each with its own partial tiles, replayed in turn
    with eager calls between; and either product against the oracle."""
    say(f"[mxfp4 split graphs] H={H} F={F} {counts}")
    E, R = len(counts), sum(counts)
    q, s, w = _experts(E, F, H, H + F)
    offs = _offsets(counts).to(dev())
    g = torch.Generator(device=dev()).manual_seed(R)
    x, dy = (torch.randn(2, R, H, device=dev(), generator=g).bfloat16() for _ in range(2))
    hgu, y, p = _forward(x[0], q, s, offs, F)
    tiles = lambda bm: sum(-(-c // bm) for c in counts)  # noqa: E731
    assert p.tiles() == tiles(fwd) and p.split() == split[0]
    dx, p = _backward(dy[0], hgu, q, s, offs, F)
    assert p.tiles() == tiles(dxp) and p.split() == split[1]
    rh, ry, th, ty = OX.swiglu_fwd(x[0], w, offs.tolist())
    _inside(hgu, rh, th, "hgu")
    _inside(y, ry, ty, "y")
    rx, tx = OX.swiglu_bwd(dy[0], hgu, w, offs.tolist())
    _inside(dx, rx, tx, "dxp")

    def step(t, d):
        h, o = ops.swiglu_forward_mxfp4(t, q, s, offs)
        return h, o, ops.swiglu_backward_mxfp4(d, h, q, s, offs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        buf = [(x[k].clone(), dy[k].clone()) for k in range(2)]
        assert all(torch.equal(a, b) for a, b in zip(step(*buf[0]), (hgu, y, dx)))
    side.synchronize()
    graphs, outs = [], []
    for b in buf:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append(step(*b))
        graphs.append(gr)
    for i in range(3):
        for k in (1, 0):
            buf[k][0].copy_(x[k] * (i + 1))
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], step(*buf[k]))), (i, k)


@pytest.mark.parametrize("H,F,E,sizes", [
    (544, 1056, 2, (1, 16, 17, 33, 40)),           # few blocks: eight waves share a weight row's units, at any rows
    (2048, 2048, 8, (8, 16, 17, 33, 40)),          # four waves, from 8 rows on
    (1024, 1024, 16, (16, 17, 33, 40)),            # two waves, from 16 rows on
], ids=["8-waves", "4-waves", "2-waves"])
def test_a_rows_bits_within_one_few_row_form(H, F, E, sizes):
    """With as many waves to a weight row a row's sums run in one order, whatever rows are beside it.  (How many waves there are
    goes by the batch's rows: between those a row's last bits may differ.)"""
    say(f"[mxfp4 row bits] H={H} F={F}")
    q, s, _ = _experts(E, F, H, 29)
    x = torch.randn(sizes[-1], H, device=dev(), generator=torch.Generator(device=dev()).manual_seed(1)).bfloat16()

    def run(n):
        offs = _offsets([0] * (E - 1) + [n]).to(dev())
        return ops.swiglu_forward_mxfp4(x[:n], q, s, offs)

    hgu, y = run(sizes[-1])
    for n in sizes[:-1]:
        a, b = run(n)
        assert torch.equal(a, hgu[:n]) and torch.equal(b, y[:n]), n
