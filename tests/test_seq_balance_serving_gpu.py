"""The sequences of the balance loss in the layer's other forwards: e4m3 and 4-bit experts see the batch as ``forward`` does, and a
forward that records no gradient launches nothing for the loss until it is read."""

from __future__ import annotations

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import _lib
from pkg.distributed import build_topology
from pkg.distributed.moe_layer import DistributedMoELayer
from pkg.models import ToyMoEBlock

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


def _kernels(f):
    torch.cuda.synchronize()
    _lib.prof_enable(True)
    try:
        f()
    finally:
        _lib.prof_enable(False)
    return set(_lib.prof_summary())


@pytest.mark.parametrize("shape", [(Bn, S, H), (57, H), (1, 1, H), (0, S, H), (2, 0, H)], ids=str)
def test_serving_forms_the_loss_when_it_is_read(shape):
    say(f"[seq balance serving] {shape}")
    layer = _layer(check_numerics=False)
    block = ToyMoEBlock(H, F, E, K, build_topology(), dtype=B, layout="routed", seq_balance_coef=0.5).to(dev())
    x = torch.randn(shape, device=dev()).to(B)
    n = x.numel() // H
    for f, r in ((layer.forward, layer.router), (layer.forward_fp8, layer.router), (layer.forward_mxfp4, layer.router),
                 (layer.router, layer.router), (block, block.moe.router)):
        if n == 0 and f == layer.forward_fp8:
            continue

        def serve():
            with torch.no_grad():
                f(x)

        names = _kernels(serve)
        assert not any("balance" in k for k in names) and (n == 0 or names), names
        got = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
        assert not got[0].requires_grad
        if f != layer.forward_fp8:  # formed at once where a gradient is recorded
            f(x)
            assert r._seq_later is None and r.last_seq_balance_loss.requires_grad
            want = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        rows = shape[0] if len(shape) == 3 and shape[0] > 0 else 1
        assert got[1].shape == (rows, E) and int(got[2][-2]) == n and int(got[1].sum()) == n * K


def test_read_after_replays_of_a_decode_graph():
    """Each read is of the logits that the last replay left."""
    say("[seq balance decode graph]")
    layer = _layer(check_numerics=False)
    r, side = layer.router, torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            buf = _tokens(1)
            layer.forward_mxfp4(buf)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = layer.forward_mxfp4(buf)
        held = r._seq_later
        for i in range(4):
            buf.copy_(_tokens(10 + i))
            g.replay()
            torch.cuda.synchronize()
            r._seq_later = held
            got = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
            assert torch.equal(layer.forward_mxfp4(buf), out)  # eager
            want = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_values_of_the_last_forward_can_be_set():
    say("[seq balance set]")
    layer = _layer(check_numerics=False)
    r = layer.router
    with torch.no_grad():
        layer(_tokens())
    counts = r.last_seq_counts
    r.last_seq_balance_loss = None
    assert r.last_seq_balance_loss is None and torch.equal(r.last_seq_counts, counts)
    with torch.no_grad():
        layer(_tokens())
        r.seq_balance_coef = 7.0  # the loss is that of the forward
        a = r.last_seq_balance_loss
        r.seq_balance_coef = 0.5
        layer(_tokens())
        assert torch.equal(r.last_seq_balance_loss, a)
        r.seq_balance_coef = 0.0
        layer(_tokens())
    assert r.last_seq_balance_loss is None and r.last_seq_counts is None and r.last_seq_tokens is None


def test_read_on_another_stream_than_the_forwards():
    """The read's kernels wait behind other work while later forwards, on their own stream, take and fill new memory."""
    say("[seq balance streams]")
    layer = _layer(check_numerics=False)
    r, side = layer.router, torch.cuda.Stream()
    xs = [_tokens(20 + i) for i in range(8)]
    with torch.no_grad():
        layer.forward_mxfp4(xs[0])
        want = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.forward_mxfp4(xs[0])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(20_000_000)
        got = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
        with torch.cuda.stream(side):
            for x in xs[1:]:
                layer.forward_mxfp4(x)
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_served_in_inference_mode_read_outside():
    say("[seq balance inference mode]")
    layer = _layer(check_numerics=False)
    r, x = layer.router, _tokens(40)
    with torch.inference_mode():
        layer.forward_mxfp4(x)
    got = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
    with torch.inference_mode():
        inside = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
    layer.forward_mxfp4(x)  # a gradient is recorded: formed at once
    want = r.last_seq_balance_loss, r.last_seq_counts, r.last_seq_tokens
    assert want[0].requires_grad and not got[0].requires_grad
    assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(got, want, inside))
