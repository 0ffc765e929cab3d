"""oracle/balance.py against the whole-batch losses of oracle/router.py and central differences, and the argument checks of
the entry points (CPU only)."""

from __future__ import annotations

import pytest
import torch

from oracle import balance as OB
from oracle import router as OR

from moe_mi355 import _lib, ops

pytestmark = pytest.mark.cpu


def _case(seed, N=23, E=6, K=2):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(N, E, generator=g, dtype=torch.float64)
    idx = logits.topk(K, -1).indices
    offs = torch.tensor([2, 2, 9, 10, 20])
    mask = torch.rand(N, generator=g) < 0.7
    return logits, idx, offs, mask


def test_one_sequence_is_the_whole_batch_loss():
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(40, 16, generator=g), torch.randn(16, 6, generator=g) * 0.3
    ref = OR.router_full(x, w, 2, grad_w=torch.zeros(40, 2), alpha=0.01, beta=1e-3)
    fwd = OR.route_fwd(x, w, 2)
    out = OB.balance(fwd["logits"], fwd["idx"], balance_coef=0.01, z_coef=1e-3)
    assert abs(float(out["balance"]) - float(ref["aux"])) < 1e-12
    assert abs(float(out["z"]) - float(ref["z"])) < 1e-12
    assert float((x.double() @ w.double() - fwd["logits"]).abs().max()) < 1e-6
    assert float((out["dlogits"] @ w.double().T - ref["dX"]).abs().max()) < 1e-9


def test_gradient_against_differences():
    logits, idx, offs, mask = _case(0)
    out = OB.balance(logits, idx, offs, mask, 0.7, 0.3, 1.5, -0.5)

    def f(t):
        o = OB.balance(t, idx, offs, mask, 0.7, 0.3)
        return 1.5 * float(o["balance"]) - 0.5 * float(o["z"])

    for t in range(logits.shape[0]):
        for e in (0, 3):
            h = torch.zeros_like(logits)
            h[t, e] = 1e-5
            assert abs((f(logits + h) - f(logits - h)) / 2e-5 - float(out["dlogits"][t, e])) < 1e-8


def test_left_out_tokens_do_not_matter():
    logits, idx, offs, mask = _case(1)
    a = OB.balance(logits, idx, offs, mask, 1.0, 1.0)
    out = ~mask
    out[:2] = True
    out[20:] = True
    logits[out] = float("nan")
    b = OB.balance(logits, idx, offs, mask, 1.0, 1.0)
    assert all(torch.equal(a[k], b[k]) for k in a)
    assert a["tokens"][0] == 0 and a["tokens"][-1] <= 3


def test_c_abi_refusals():
    lib = _lib.load()
    f = 4096  # an aligned address that no call below reads
    for N, E, K, S in ((0, 8, 2, 1), (4, 300, 2, 1), (4, 8, 9, 1), (4, 64, 33, 1), (4, 8, 0, 1), (4, 8, 2, 0)):
        assert lib.moe_balance_fwd(f, f, f, None, N, E, K, S, 1.0, 0.0, f, f, f, f, f, f, 1 << 20, None) == -1
        assert "bad shape" in _lib.last_error()
        assert lib.moe_balance_bwd(f, f, f, f, None, None, None, N, E, K, S, 1.0, 0.0, f, None) == -1
    assert lib.moe_balance_fwd(f, f, None, None, 4, 8, 2, 3, 1.0, 0.0, f, f, f, f, f, f, 1 << 20, None) == -1  # S needs offsets
    assert lib.moe_balance_fwd(f, f, f, None, 4, 8, 2, 3, 1.0, 0.0, f, f, f, f, f, f, 8, None) == -2
    assert lib.moe_balance_fwd(None, f, f, None, 4, 8, 2, 3, 1.0, 0.0, f, f, f, f, f, f, 1 << 20, None) == -1
    assert lib.moe_balance_bwd(f, f, None, f, None, None, None, 4, 8, 2, 3, 1.0, 0.0, f, None) == -1
    assert lib.moe_balance_fwd_workspace(0, 8, 1) == 0 and lib.moe_balance_fwd_workspace(100, 8, 4) > 0


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        ops.balance_loss_forward(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64))
