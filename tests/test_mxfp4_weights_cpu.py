"""The layer's 4-bit weights as buffers: taken, moved and kept out of the state_dict (CPU only: nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer

pytestmark = pytest.mark.cpu

H, F, E = 64, 96, 3


def _layer():
    return DistributedMoELayer(H, F, E, 2, build_topology(device_type="cpu"), dtype=torch.bfloat16)


def _weights(E=E, F=F, H=H):
    g = torch.Generator().manual_seed(1)
    shapes = ((E, F, H), (E, F, H), (E, H, F))
    return ([torch.randint(0, 256, (*s[:2], s[2] // 2), dtype=torch.uint8, generator=g) for s in shapes],
            [torch.randint(100, 130, (*s[:2], s[2] // 32), dtype=torch.uint8, generator=g) for s in shapes])


def test_they_move_with_the_layer_and_stay_bytes():
    layer = _layer()
    q, s = _weights()
    got = layer.load_mxfp4(q, s)
    assert all(a is b or torch.equal(a, b) for a, b in zip(got[0] + got[1], q + s))
    layer.float()
    held = {n: t for n, t in layer.named_buffers() if "mxfp4" in n}
    assert len(held) == 6 and all(t.dtype == torch.uint8 for t in held.values())
    layer.to("meta")
    assert all(t.device.type == "meta" for n, t in layer.named_buffers() if "mxfp4" in n)


def test_state_dict_keeps_the_references_keys():
    a, b = _layer(), _layer()
    keys = list(a.state_dict())
    a.load_mxfp4(*_weights())
    assert list(a.state_dict()) == keys
    b.load_state_dict(a.state_dict())  # strict, both ways
    a.load_state_dict(b.state_dict())
    assert a.mxfp4_gate is not None and b.mxfp4_gate is None


def test_taken_in_inference_mode_they_can_be_trained_around():
    layer = _layer()
    with torch.inference_mode():
        q, s = _weights()
        got = layer.load_mxfp4(q, s)
    assert not any(t.is_inference() for t in got[0] + got[1])
    assert all(torch.equal(a, b) for a, b in zip(got[0] + got[1], q + s))


def test_dropped_full_width_weights():
    layer = _layer()
    layer.load_mxfp4(*_weights())
    layer.w_gate = layer.w_up = layer.w_down = None
    assert [n for n, _ in layer.named_parameters()] == ["router.gate_w"]
    assert list(layer.state_dict()) == ["router.gate_w"]
    layer.load_state_dict(layer.state_dict())
    with pytest.raises(RuntimeError, match="dropped"):
        layer.quantize_mxfp4()
    with pytest.raises(RuntimeError, match="dropped"):
        layer.experts[0](torch.zeros(1, H))


def test_refusals():
    layer = _layer()
    q, s = _weights()
    for bad in (([q[0].int(), q[1], q[2]], s), ([q[0].transpose(0, 1), q[1], q[2]], s)):
        with pytest.raises(TypeError):
            layer.load_mxfp4(*bad)
    for bad in ((q, [s[0], s[1], s[2][:, :, :1].contiguous()]), _weights(E=2), _weights(F=32), _weights(H=32), (q[:2], s)):
        with pytest.raises(ValueError):
            layer.load_mxfp4(*bad)
    assert layer.mxfp4_gate is None
    with pytest.raises(RuntimeError, match="load_mxfp4"):
        layer.forward_mxfp4(torch.zeros(1, H, dtype=torch.bfloat16))
