"""The balance loss of sequences and the z-loss over valid tokens on the GPU against oracle/balance.py: counts equal,
probabilities, losses and gradients within bounds derived from fp32.

A probability is exp(l - m) / sum: the difference is off by 2^-24 |l - m|, exp by 2 ulps, the sum of E terms by E 2^-24, the
division by one: relative (E + 8 + |l - m|) 2^-24, with |l - m| <= 40 taken in (smaller probabilities are below 2^-57).
``lse`` is off by 2^-24 (2 |lse| + E + 8)."""

from __future__ import annotations

import threading

import pytest
import torch

from gpu_util import dev, say

from moe_mi355 import ops
from oracle import balance as OB

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BC, ZC, GB, GZ = 0.01, 1e-3, 1.5, -0.75


def _case(N, E, K, lengths, masked, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + N + 31 * E)
    logits = torch.randn(N, E, generator=g) * spread
    idx = logits.topk(K, -1).indices
    offs = None
    if lengths is not None:
        offs = torch.tensor([lengths[0]] + list(lengths[0] + torch.tensor(lengths[1]).cumsum(0)))
        assert int(offs[-1]) <= N
    mask = None
    if masked:
        mask = torch.rand(N, generator=g) < 0.6
    out = torch.zeros(N, dtype=torch.bool) if offs is None else \
        (torch.arange(N) < offs[0]) | (torch.arange(N) >= offs[-1])
    if mask is not None:
        out |= ~mask
    logits[out] = torch.tensor([float("nan"), float("inf"), -float("inf")])[torch.arange(int(out.sum())) % 3].unsqueeze(1)
    return logits, idx, offs, mask


def _run(logits, idx, offs, mask):
    d = dev()
    lg = logits.to(d)
    o, m = (None if t is None else t.to(d) for t in (offs, mask))
    f = ops.balance_loss_forward(lg, idx.to(d), o, m, BC, ZC)
    g = ops.balance_loss_backward(lg, f[2], f[3], idx.shape[1], o, m, torch.tensor(GB, device=d), torch.tensor(GZ, device=d),
                                  BC, ZC)
    return f, g


RAGGED = [5, 0, 1, 17, 0, 0, 64, 3, 200, 1, 1, 1, 33]
SHAPES = [
    (1, 1, 1, None, False),
    (1, 8, 2, (0, [1]), True),
    (7, 5, 5, (0, [7]), False),                       # every expert chosen
    (1000, 8, 2, (3, RAGGED), True),                  # tokens before and behind the sequences
    (1000, 16, 4, None, True),
    (333, 17, 3, (0, RAGGED), False),
    (2000, 64, 6, (100, [700, 0, 900, 299]), True),
    (300, 33, 32, (0, [1] * 300), False),             # one token each
    (900, 128, 8, (0, [0] * 100 + [3] * 200 + [0] * 300), True),
    (500, 256, 8, (0, [100, 400]), False),
    (70000, 8, 1, (1000, [20000, 1, 40000]), True),   # longer runs
    (5, 8, 2, (0, [0, 0, 0]), False),                 # no sequence has a token
    (40, 200, 2, (0, [40] + [0] * 5000), True),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"N{s[0]}-E{s[1]}-K{s[2]}")
@pytest.mark.parametrize("spread", [1.0, 8.0])
def test_against_the_oracle(shape, spread):
    N, E, K, lengths, masked = shape
    say(f"[balance] {N} {E} {K} masked={masked} spread={spread}")
    logits, idx, offs, mask = _case(N, E, K, lengths, masked, spread=spread)
    (balance, z, counts, tokens, mean_prob), d = _run(logits, idx, offs, mask)
    ref = OB.balance(logits, idx, offs, mask, BC, ZC, GB, GZ)
    assert torch.equal(counts.cpu(), ref["counts"]) and torch.equal(tokens.cpu(), ref["tokens"])
    rel = (E + 8 + 40) * U
    n_max = max(1, int(ref["tokens"][:-2].max()))
    run = 64  # tokens that a wave adds up in fp32 before the sums go on in 64 bits
    assert float((mean_prob.cpu().double() - ref["mean_prob"]).abs().max()) <= (rel + min(n_max, run) * U) * 1.0
    assert abs(float(balance) - float(ref["balance"])) <= (rel + (min(n_max, run) + 2) * U) * abs(float(ref["balance"])) + 1e-30
    valid = torch.nan_to_num(ref["dlogits"]).abs().sum(1) > 0
    big = 1.0 if not bool(valid.any()) else float(torch.logsumexp(logits[valid].double(), 1).abs().max())
    lse_off = (2 * big + E + 8) * U
    n_all = max(1, int(ref["tokens"][-2]))
    assert abs(float(z) - float(ref["z"])) <= ZC * (2 * big * lse_off + (min(n_all, run) + 4) * U * big * big)
    # gradient: cb p (f - pf) + cz lse p, term by term; f and pf are at most E
    used, n = max(1, int(ref["tokens"][-1])), ref["tokens"][:-2].clamp(min=1).double()
    per = torch.zeros(N, dtype=torch.float64)
    bounds = [0, N] if offs is None else offs.tolist()
    for s in range(len(bounds) - 1):
        per[bounds[s]:bounds[s + 1]] = 1.0 / float(n[s])
    p = torch.softmax(torch.where(valid.unsqueeze(1), logits, torch.zeros(())).double(), 1)
    cb = abs(GB) * BC / used * per.unsqueeze(1)
    cz = abs(GZ) * ZC * 2 / n_all
    tol = p * (cb * E * (2 * rel + (E + 8) * U) + cz * (big * (rel + 6 * U) + lse_off)) + 1e-40
    off = (d.cpu().double() - ref["dlogits"]).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    left = torch.ones(N, dtype=torch.bool)
    for s in range(len(bounds) - 1):
        left[bounds[s]:bounds[s + 1]] = False
    if mask is not None:
        left |= ~mask
    assert bool((d.cpu()[left] == 0).all())


@pytest.mark.parametrize("shape", [
    (1024, 8, 8, (0, [64] * 16), False),                  # the most that one block takes, and one more of each
    (1025, 8, 2, (1, [64] * 16), True),
    (1024, 7, 3, (0, [0, 1024] + [0] * 14), True),
    (1000, 8, 2, (0, [50] * 17), True),
    (512, 16, 16, (12, [1, 0, 499]), True),
    (128, 64, 32, (0, [8] * 16), False),
    (129, 64, 6, (0, [129]), True),
    (128, 65, 6, (0, [100, 28]), True),
    (2, 3, 1, (0, [0, 2]), False),
], ids=lambda s: f"N{s[0]}-E{s[1]}-K{s[2]}-S{len(s[3][1])}")
def test_small_batches(shape):
    test_against_the_oracle(shape, 2.0)


@pytest.mark.parametrize("N,E,lengths,one", [
    (384, 8, None, True), (385, 8, None, False), (1000, 8, None, False),  # one sequence: 8 tokens a step
    (768, 8, [700, 68], True), (769, 8, [700, 69], False),
    (1024, 8, [256] * 4, True), (1024, 8, [64] * 16, True), (1024, 8, [60] * 17, False), (1025, 8, [64] * 16, False),
    (192, 16, None, True), (193, 16, None, False), (48, 64, None, True), (49, 64, None, False), (128, 64, [64, 64], False),
    (96, 64, [1, 95], True), (20, 65, None, False),
], ids=lambda v: str(v)[:24])
def test_which_form_a_small_batch_takes(N, E, lengths, one):
    """One block only where its waves' sequences are short on average; either form against the oracle."""
    from moe_mi355 import _lib

    logits, idx, offs, mask = _case(N, E, min(E, 4), None if lengths is None else (0, lengths), True, seed=7)
    torch.cuda.synchronize()
    _lib.prof_enable(True)
    try:
        f, _ = _run(logits, idx, offs, mask)
    finally:
        _lib.prof_enable(False)
    names = set(_lib.prof_summary())
    assert ("k_balance_one" in names) == one and ("k_balance_fwd" in names) != one, names
    test_against_the_oracle((N, E, min(E, 4), None if lengths is None else (0, lengths), True), 2.0)
    ref = OB.balance(logits, idx, offs, mask, BC, ZC, GB, GZ)
    assert torch.equal(f[2].cpu(), ref["counts"]) and torch.equal(f[3].cpu(), ref["tokens"])


def test_masks_of_the_lowest_value_and_minus_infinity():
    """Experts closed to a token by the type's lowest value or by -inf have probability 0; all closed by the lowest value is
    a uniform token."""
    N, E = 64, 8
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(N, E, generator=g)
    logits[:, 3] = -float("inf")
    logits[5:9, 4:] = torch.finfo(torch.float32).min
    idx = logits.topk(2, -1).indices
    ref = OB.balance(logits, idx, None, None, BC, ZC, GB, GZ)
    (balance, z, counts, _, mean_prob), d = _run(logits, idx, None, None)
    assert float(mean_prob[0, 3]) == 0.0 and torch.equal(counts.cpu(), ref["counts"])
    assert abs(float(balance) - float(ref["balance"])) <= 200 * U * float(ref["balance"])
    assert abs(float(z) - float(ref["z"])) <= 200 * U * float(ref["z"])
    assert float((d.cpu().double() - ref["dlogits"]).abs().max()) <= 200 * U * float(ref["dlogits"].abs().max()) * E
    logits[7] = torch.finfo(torch.float32).min
    (balance, z, _, _, mean_prob), d = _run(logits, idx, None, None)
    p = torch.softmax(logits.double(), 1).mean(0)
    assert float((mean_prob[0].cpu().double() - p).abs().max()) <= 200 * U


def test_ids_out_of_range_count_for_none():
    logits = torch.randn(50, 8)
    idx = torch.randint(0, 8, (50, 3))
    idx[::7, 1] = -1
    idx[::5, 2] = 8
    idx[3, 0] = 1 << 40
    (_, _, counts, _, _), _ = _run(logits, idx, None, None)
    assert torch.equal(counts.cpu(), OB.balance(logits, idx)["counts"])


def test_same_expert_twice_counts_twice():
    idx = torch.tensor([[2, 2], [1, 2]])
    (_, _, counts, _, _), _ = _run(torch.randn(2, 4), idx, None, None)
    assert counts.cpu().tolist() == [[0, 1, 3, 0]]


def test_views_int32_offsets_and_empty():
    logits, idx, offs, mask = _case(400, 24, 4, (0, [100, 250, 50]), True)
    want = _run(logits, idx, offs, mask)
    d = dev()
    wide = torch.zeros(400, 48, device=d)
    wide[:, ::2] = logits.to(d)
    ids = idx.to(d).T.contiguous().T
    f = ops.balance_loss_forward(wide[:, ::2], ids, offs.int().to(d), mask.reshape(20, 20).to(d), BC, ZC)
    assert all(torch.equal(a, b) for a, b in zip(f, want[0]))
    b = ops.balance_loss_backward(wide[:, ::2], f[2], f[3], 4, offs.int().to(d), mask.to(d), torch.tensor(GB, device=d),
                                  torch.tensor(GZ, device=d).double(), BC, ZC)
    assert torch.equal(b, want[1])
    f = ops.balance_loss_forward(wide[:0], ids[:0], None, None)
    assert float(f[0]) == 0 and f[2].shape == (1, 48) and f[3].tolist() == [0, 0, 0]
    assert ops.balance_loss_backward(wide[:0], f[2], f[3], 4).shape == (0, 48)


def test_same_bits_in_graphs_streams_and_threads():
    say("[balance graph]")
    logits, idx, offs, mask = _case(3000, 64, 6, (10, [900, 1, 0, 1500]), True)
    want = [t.clone() for f in [_run(logits, idx, offs, mask)] for t in (*f[0], f[1])]
    d = dev()
    lg, ix, of, mk = (t.to(d) for t in (logits, idx, offs, mask))
    gb, gz = torch.tensor(GB, device=d), torch.tensor(GZ, device=d)

    def step(t):
        f = ops.balance_loss_forward(t, ix, of, mk, BC, ZC)
        return (*f, ops.balance_loss_backward(t, f[2], f[3], 6, of, mk, gb, gz, BC, ZC))

    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        assert same(step(lg), want)
        buf = lg.clone()
    side.synchronize()
    for _ in range(2):  # two graphs whose replays alternate
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(buf)
        graphs.append((g, out))
    for i in range(4):
        buf.copy_(lg * (1 + i))
        eager = [t.clone() for t in step(buf)]
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            assert same(out, eager)
    fails = []

    def work(k):
        try:
            for _ in range(20):
                if not same(step(lg), want):
                    fails.append(k)
        except Exception as e:  # raised again by the test's own thread
            fails.append(e)

    ts = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not fails, fails


def test_refusals():
    d = dev()
    lg, idx = torch.randn(10, 8, device=d), torch.zeros(10, 2, dtype=torch.int64, device=d)
    f = ops.balance_loss_forward
    with pytest.raises(TypeError):
        f(lg.bfloat16(), idx)
    with pytest.raises(ValueError):
        f(lg, idx.int())
    with pytest.raises(ValueError):
        f(lg, idx[:5])
    with pytest.raises(ValueError):
        f(lg, idx, torch.tensor([0.0, 10.0], device=d))
    with pytest.raises(ValueError):
        f(lg, idx, torch.tensor([0], device=d))
    with pytest.raises(ValueError):
        f(lg, idx, None, torch.ones(9, dtype=torch.bool, device=d))
    with pytest.raises(ValueError):
        f(lg, idx, None, torch.ones(10, device=d))
    with pytest.raises(RuntimeError):
        f(lg, idx.cpu())
    with pytest.raises(ValueError):
        f(torch.randn(4, 300, device=d), idx[:4])
    with pytest.raises(ValueError):
        f(torch.randn(10, 1, device=d), idx)
    out = f(lg, idx)
    with pytest.raises(ValueError):
        ops.balance_loss_backward(lg, out[2], out[3][:2], 2)
    with pytest.raises(ValueError):
        ops.balance_loss_backward(lg, out[2][:, :4], out[3], 2)
    with pytest.raises(ValueError):
        ops.balance_loss_backward(lg, out[2], out[3], 0)


@pytest.mark.parametrize("N,E,K,lengths", [
    (66000, 8, 2, [40000, 0, 25990]), (66000, 16, 4, [30000, 1, 0, 35000]), (66001, 15, 4, None),
    (65700, 32, 4, [1000] * 65), (65701, 30, 8, [65700]), (33000, 64, 6, [32999]), (33001, 62, 6, [100] * 330),
    (32900, 128, 8, [16000, 16000, 1]), (32901, 126, 32, None), (16500, 256, 8, [5] * 3300), (16501, 254, 3, [16000, 501]),
], ids=lambda v: str(v)[:24])
def test_long_batches(N, E, K, lengths):
    """Batches that give every lane group several tokens: each number of lanes a token, with and without 16-byte loads."""
    test_against_the_oracle((N, E, K, None if lengths is None else (0, lengths), True), 2.0)
