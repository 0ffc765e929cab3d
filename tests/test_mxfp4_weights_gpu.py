"""A layer served from 4-bit weights that were moved, handed in, or are the only ones it holds."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer

pytestmark = pytest.mark.gpu

B = torch.bfloat16
H, F, E, K = 128, 96, 4, 2


def _layer(seed):
    torch.manual_seed(seed)
    return DistributedMoELayer(H, F, E, K, build_topology(), dtype=B, layout="routed").to(dev())


def test_moved_handed_in_and_alone():
    say("[mxfp4 weights]")
    layer = _layer(0)
    q, s = layer.quantize_mxfp4()
    x = torch.randn(9, H, device=dev()).to(B)
    with torch.no_grad():
        want = layer.forward_mxfp4(x)
        layer.cpu()
        assert not any(t.is_cuda for t in layer.buffers())
        layer.to(dev())
        assert torch.equal(layer.forward_mxfp4(x), want)
        other = _layer(1)
        other.router.load_state_dict(layer.router.state_dict())
        other.load_mxfp4([t.cpu() for t in q], [t.cpu() for t in s])  # from the host, as a file gives them
        assert torch.equal(other.forward_mxfp4(x), want)
        before = other.forward(x)
        other.w_gate = other.w_up = other.w_down = None
        assert torch.equal(other.forward_mxfp4(x), want) and not torch.equal(before, want)
        with pytest.raises(RuntimeError, match="dropped"):
            other.forward(x)
        with pytest.raises(NotImplementedError):
            other.forward_fp8(x)
    y = x.clone().requires_grad_(True)  # still differentiable in the tokens and the gate
    a = torch.autograd.grad(other.forward_mxfp4(y).float().square().sum(), [y, other.router.gate_w])
    b = torch.autograd.grad(layer.forward_mxfp4(y).float().square().sum(), [y, layer.router.gate_w])
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_quantized_and_served_in_inference_mode_then_trained():
    say("[mxfp4 weights inference mode]")
    layer = _layer(2)
    x = torch.randn(5, H, device=dev()).to(B)
    with torch.inference_mode():
        layer.quantize_mxfp4()
        want = layer.forward_mxfp4(x)
    y = x.clone().requires_grad_(True)
    out = layer.forward_mxfp4(y)
    assert torch.equal(out, want)
    out.float().square().sum().backward()
    assert float(y.grad.abs().max()) > 0 and float(layer.router.gate_w.grad.abs().max()) > 0
