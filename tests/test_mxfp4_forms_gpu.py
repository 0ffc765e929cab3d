"""The forms of the 4-bit experts' products, each shown to be the one that ran: through the C ABI, whose caller owns the
workspace, where the row tiles and the partial tiles of a split last round can be seen."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say
from test_mxfp4_gpu import _inside, _offsets

from moe_mi355 import _lib
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
