"""The sequences of the balance loss in the layer's other forwards: e4m3 and 4-bit experts see the batch as ``forward`` does."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer

pytestmark = pytest.mark.gpu

B = torch.bfloat16
Bn, S, H, F, E, K = 3, 40, 256, 128, 8, 2


def _layer(**kw):
    torch.manual_seed(5)
    layer = DistributedMoELayer(H, F, E, K, build_topology(), dtype=B, layout="routed", seq_balance_coef=0.5, **kw).to(dev())
    layer.quantize_mxfp4()
    return layer


def _tokens(seed=0):
    return torch.randn(Bn, S, H, device=dev(), generator=torch.Generator(device=dev()).manual_seed(seed)).to(B)


@pytest.mark.parametrize("how", ["rows", "mask", "offsets", "both"])
def test_every_forward_has_the_same_sequences(how):
    say(f"[seq balance forwards] {how}")
    layer, x = _layer(z_loss_coef=1e-2), _tokens()
    kw = {}
    if how in ("mask", "both"):
        kw["token_mask"] = torch.arange(S, device=dev()) < torch.tensor([[40], [0], [7]], device=dev())
    if how in ("offsets", "both"):
        kw["seq_offsets"] = torch.tensor([0, 11, 11, 100, 117], device=dev())
    r, want = layer.router, None
    with torch.no_grad():
        for f in (layer.forward, layer.forward_fp8, layer.forward_mxfp4):
            assert f(x, **kw).shape == x.shape
            got = (r.last_seq_balance_loss, r.last_z_loss, r.last_seq_counts, r.last_seq_tokens)
            assert got[2].shape == (4 if "seq_offsets" in kw else Bn, E)
            want = want or got
            assert all(torch.equal(a, b) for a, b in zip(got, want)), f.__name__
