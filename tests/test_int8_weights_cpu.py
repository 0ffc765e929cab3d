"""The layer's int8 weights as buffers: taken, moved, left alone by a change of dtype and kept out of the state_dict; refusals of
the int8 and norm operators on CPU tensors and through the C ABI (CPU only: nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from moe_mi355 import _lib, ops
from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer
from pkg.models import RMSNorm, ToyMoEBlock

pytestmark = pytest.mark.cpu

H, F, E = 64, 96, 3


def _layer():
    return DistributedMoELayer(H, F, E, 2, build_topology(device_type="cpu"), dtype=torch.bfloat16)


def _weights(E=E, F=F, H=H):
    g = torch.Generator().manual_seed(1)
    shapes = ((E, F, H), (E, F, H), (E, H, F))
    return ([torch.randint(-127, 128, s, dtype=torch.int8, generator=g) for s in shapes],
            [torch.rand(s[:2], generator=g) for s in shapes])


def test_they_move_with_the_layer_and_keep_their_types():
    layer = _layer()
    q, s = _weights()
    got = layer.load_int8(q, s)
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got[0] + got[1], q + s))
    for change in (layer.float, layer.bfloat16, layer.double):
        change()
        got = layer._int8_weights()
        assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got[0] + got[1], q + s))
    layer.to("meta")
    assert all(t.device.type == "meta" for n, t in layer.named_buffers() if "int8" in n)


def test_state_dict_keeps_the_references_keys():
    a, b = _layer(), _layer()
    keys = list(a.state_dict())
    a.load_int8(*_weights())
    assert list(a.state_dict()) == keys
    b.load_state_dict(a.state_dict())
    assert a.int8_gate is not None and b.int8_gate is None


def test_dropped_full_width_weights():
    layer = _layer()
    layer.load_int8(*_weights())
    layer.w_gate = layer.w_up = layer.w_down = None
    assert layer._int8_weights()[0][0].shape == (E, F, H)
    with pytest.raises(RuntimeError, match="dropped"):
        layer.quantize_int8()


def test_load_refuses():
    layer = _layer()
    q, s = _weights()
    with pytest.raises(ValueError, match="up must be"):
        layer.load_int8((q[0], q[2], q[2]), s)
    with pytest.raises(ValueError, match="scales"):
        layer.load_int8(q, (s[0], s[1], s[0]))
    with pytest.raises(TypeError, match="int8"):
        layer.load_int8([t.float() for t in q], s)
    with pytest.raises(TypeError, match="float32"):
        layer.load_int8(q, [t.double() for t in s])
    assert layer.int8_gate is None
    with pytest.raises(RuntimeError, match="quantize_int8"):
        layer.forward_int8(torch.zeros(2, H, dtype=torch.bfloat16))
    layer.load_int8(q, s)
    with pytest.raises(TypeError, match="bfloat16"):
        layer.forward_int8(torch.zeros(2, H))
    with pytest.raises(ValueError, match="rank"):
        layer.forward_int8(torch.zeros(H, dtype=torch.bfloat16))


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, H), torch.ones(H)
    q, s = torch.zeros(2, H, dtype=torch.int8), torch.ones(2)
    for call in (lambda: ops.quant_rows_int8(x), lambda: ops.dequant_rows(q, s), lambda: ops.matmul_int8(q, s, q, s),
                 lambda: ops.rmsnorm_quant(x, w, 1e-5), lambda: ops.rmsnorm_residual_forward(x, x, w, 1e-5),
                 lambda: ops.rmsnorm_residual_backward(x, w, s, x, x), lambda: RMSNorm(H)(x, residual=x)):
        with pytest.raises(RuntimeError, match="AMD Instinct"):
            call()
    with pytest.raises(ValueError, match="residual must be"):
        RMSNorm(H)(x, residual=x[:1])
    with pytest.raises(ValueError, match="residual must be"):
        RMSNorm(H).quantized(x, residual=x[:1])
    block = ToyMoEBlock(H, F, E, 2, build_topology(device_type="cpu"), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="rank"):
        block.forward_int8(torch.zeros(H, dtype=torch.bfloat16))


def test_c_abi_refuses_before_it_launches():
    lib = _lib.load()
    P = 16  # a pointer that is aligned and never used

    def bad(rc, text, code=-1):
        assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())

    bad(lib.moe_quant_rows_int8(P, 1, 4, 40, 40, P, P, None), "bad arguments")
    bad(lib.moe_quant_rows_int8(P, 1, 4, 48, 47, P, P, None), "bad arguments")
    bad(lib.moe_quant_rows_int8(P, 3, 4, 48, 48, P, P, None), "bad arguments")
    bad(lib.moe_quant_rows_int8(8, 1, 4, 48, 48, P, P, None), "misaligned")
    assert lib.moe_quant_rows_int8(None, 1, 0, 48, 48, None, None, None) == 0
    bad(lib.moe_dequant_rows(P, 2, P, 4, 48, P, 1, None), "bad arguments")
    bad(lib.moe_dequant_rows(P, 0, None, 4, 48, P, 1, None), "null")
    mm = lib.moe_matmul_int8
    bad(mm(P, P, P, P, None, 4, 40, 8, 1, P, 1, None, 0, None), "bad arguments")
    bad(mm(P, P, P, P, None, 4, 131072, 8, 1, P, 1, None, 0, None), "bad arguments")   # the sum would not fit
    bad(mm(P, P, P, P, None, 4, 131056, 32776, 1, P, 1, None, 0, None), "bad arguments")
    bad(mm(P, P, P, P, None, 4, 32, 12, 1, P, 1, None, 0, None), "bad arguments")
    bad(mm(P, P, P, P, None, 4, 32, 8, 2, P, 1, None, 0, None), "bad arguments")       # experts without offsets
    bad(mm(P, P, P, P, P, 4, 32, 8, 1025, P, 1, None, 0, None), "bad arguments")
    bad(mm(P, P, P, P, None, 4, 32, 8, 1, P, 2, None, 0, None), "bad arguments")
    bad(mm(P, P, P, P, None, 4, 32, 8, 1, 8, 1, None, 0, None), "misaligned")
    n = lib.moe_matmul_int8_workspace(64, 14336, 4096, 1)
    assert n > 0 and lib.moe_matmul_int8_workspace(8190, 4096, 14336, 1) == 0
    bad(mm(P, P, P, P, None, 64, 14336, 4096, 1, P, 1, P, n - 1, None), "workspace", -2)
    assert mm(None, None, None, None, None, 0, 32, 8, 1, None, 1, None, 0, None) == 0
    ex = lib.moe_swiglu_fwd_int8
    bad(ex(P, P, 4, None, 1, P, P, P, P, P, P, P, 8, 32, 32, 2, P, P, 1 << 30, None), "bad arguments")  # T != R
    bad(ex(P, P, 4, P, 0, P, P, P, P, P, P, P, 8, 32, 32, 2, P, P, 1 << 30, None), "bad arguments")
    bad(ex(P, P, 8, None, 1, P, P, P, P, P, P, P, 8, 32, 40, 2, P, P, 1 << 30, None), "bad arguments")
    bad(ex(P, P, 0, P, 1, P, P, P, P, P, P, P, 8, 32, 32, 2, P, P, 1 << 30, None), "no token")
    bad(ex(P, P, 8, None, 1, P, P, P, P, P, P, None, 8, 32, 32, 2, P, P, 1 << 30, None), "null")
    bad(ex(P, P, 8, None, 1, P, P, P, P, P, P, P, 8, 32, 32, 2, P, P, 16, None), "workspace", -2)
    bad(lib.moe_rmsnorm_residual_fwd(P, None, 1, P, 0, 1e-5, 4, 64, P, P, P, None), "null")
    bad(lib.moe_rmsnorm_residual_fwd(P, P, 1, P, 0, 1e-5, 4, 60, P, P, P, None), "bad shape")
    bad(lib.moe_rmsnorm_residual_bwd(P, 1, P, 0, P, None, None, 4, 64, P, P, P, 1 << 20, None), "null")
    bad(lib.moe_rmsnorm_residual_bwd(P, 1, P, 0, P, P, P, 4, 64, P, P, P, 16, None), "workspace", -2)
    bad(lib.moe_rmsnorm_quant(P, None, 1, P, 0, 1e-5, 4, 64, 5, P, P, None, None, None), "int8 or e4m3")
    bad(lib.moe_rmsnorm_quant(P, None, 1, P, 0, 1e-5, 4, 24, 0, P, P, None, None, None), "H % 16")
    bad(lib.moe_rmsnorm_quant(P, P, 1, P, 0, 1e-5, 4, 64, 0, P, P, None, None, None), "null")  # a residual without h


def test_load_takes_three_weights_and_three_scales():
    layer = _layer()
    q, s = _weights()
    for weights, scales in ((q[:2], s[:2]), (q, s[:2]), (q[:2], s), ([*q, q[2]], s), (q, [*s, s[2]]), ([*q, q[2]], [*s, s[2]]),
                            ((), ())):
        with pytest.raises(ValueError, match="load_int8"):
            layer.load_int8(weights, scales)
        assert all(t is None for n, t in layer._buffers.items() if "int8" in n)
    got = layer.load_int8(iter(q), iter(s))
    assert all(torch.equal(a, b) for a, b in zip(got[0] + got[1], q + s))
    with pytest.raises(ValueError, match="load_int8"):  # what is there stays
        layer.load_int8(q[:2], s[:2])
    got = layer._int8_weights()
    assert all(torch.equal(a, b) for a, b in zip(got[0] + got[1], q + s))
