"""Operators of the MoE layer beside its bf16 / fp32 / e4m3 path: experts held in 4 bits, and the balance loss of sequences.

Kinds of case:

quant     a weight matrix to MXFP4 (e2m1 values, one power-of-two scale per 32) and back to the values it stands for
experts   the SwiGLU experts' forward on 4-bit weights, from one decoded token to a prefill
experts_bwd  the gradient of those experts' rows (the 4-bit weights are frozen)
balance   the balance loss and z-loss over the valid tokens of each sequence, with per-expert counts, and their gradient

The plain forms work in 32 bits (64 for long sums) and round once at the end; ``exact`` works in 64 bits.
"""

import math
import os
import sys

import numpy as np
import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(_ROOT, "composed-mixture-of-experts-engine_amd"))

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_BALANCE, _Z = 0.01, 1e-3  # the loss coefficients of the framework's configurations


def listed():
    return [
        # one expert's projection of a layer of many small experts, requantized after an update: latency counts
        {"name": "quant_one_projection", "kind": "quant", "dtype": "f32", "rows": 768, "cols": 2048},
        # a layer's stacked gate weights when a checkpoint is loaded for serving
        {"name": "quant_stacked_layer", "kind": "quant", "dtype": "bf16", "rows": 8 * 14336, "cols": 4096},
        # one decoded token: its two experts' weights are all there is to read
        {"name": "decode_one_token", "kind": "experts", "R": 2, "H": 4096, "F": 14336, "E": 8, "skew": 0.0, "keep": False},
        # a decode step of 16 sequences, every expert in use
        {"name": "decode_16_tokens", "kind": "experts", "R": 32, "H": 4096, "F": 14336, "E": 8, "skew": 0.0, "keep": False},
        # a decode step of 64 sequences over many small experts, 8 each, unevenly routed
        {"name": "decode_small_experts", "kind": "experts", "R": 512, "H": 2048, "F": 768, "E": 128, "skew": 1.1, "keep": False},
        # a chunk of a prompt beside running decodes: rows enough that neither weights nor products bound it alone
        {"name": "prefill_chunk", "kind": "experts", "R": 1002, "H": 4096, "F": 14336, "E": 8, "skew": 0.0, "keep": False},
        # a long prefill, or the forward of training a router over frozen experts
        {"name": "prefill_long", "kind": "experts", "R": 16384, "H": 4096, "F": 14336, "E": 8, "skew": 0.0, "keep": True},
        # the backward through frozen experts of a small layer, odd row counts
        {"name": "backward_small_layer", "kind": "experts_bwd", "R": 4094, "H": 1024, "F": 4096, "E": 8, "skew": 1.1},
        # the same at full size
        {"name": "backward_full_layer", "kind": "experts_bwd", "R": 16384, "H": 4096, "F": 14336, "E": 8, "skew": 0.0},
        # a small padded batch: 8 sequences
        {"name": "balance_small_batch", "kind": "balance", "N": 1000, "E": 8, "K": 2, "S": 8, "mask": True},
        # a training batch of long sequences, padding masked out
        {"name": "balance_long_sequences", "kind": "balance", "N": 65536, "E": 64, "K": 6, "S": 16, "mask": True},
        # packed short samples over many experts
        {"name": "balance_packed_samples", "kind": "balance", "N": 32768, "E": 128, "K": 8, "S": 700, "mask": False},
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quant", "experts", "experts", "experts_bwd", "balance"])
    if kind == "quant":
        cols = 32 * _logint(rng, 1, 448)
        dtype = rng.choice(["bf16", "f32"])
        most = min(8 * 14336, 8 * 14336 * 4096 // cols // (1 if dtype == "bf16" else 2))
        return {"kind": kind, "dtype": dtype, "rows": _logint(rng, 1, most), "cols": cols}
    if kind == "balance":
        N, E = _logint(rng, 1, 65536), _logint(rng, 2, 128)
        N = min(N, 65536 * 64 // E)
        return {"kind": kind, "N": N, "E": E, "K": rng.randint(1, min(8, E)), "S": _logint(rng, 1, max(1, N // 4)),
                "mask": rng.random() < 0.5}
    while True:
        c = {"kind": kind, "R": _logint(rng, 1, 16384), "H": 32 * _logint(rng, 4, 128), "F": 32 * _logint(rng, 4, 448),
             "E": _logint(rng, 1, 128), "skew": rng.choice([0.0, 1.1])}
        if kind == "experts":
            c["keep"] = rng.random() < 0.3
        room = c["E"] * (max(_counts(c)) + 1) * (2 * c["F"] + c["H"])
        if c["E"] * c["F"] * c["H"] <= 8 * 14336 * 4096 and room <= 1 << 30:
            return c


# ---- inputs ----


def _counts(case):
    """Rows of each expert, largest share first where the routing is skewed (Zipf)."""
    share = (1.0 + np.arange(case["E"])) ** -case["skew"]
    rng = np.random.default_rng([case["R"], case["E"], case["H"], case["F"]])
    return rng.multinomial(case["R"], share / share.sum()).tolist()


def _seq_lengths(case):
    """Ragged sequence lengths whose sum leaves a tail of up to a sixteenth of the tokens in no sequence; some are empty."""
    rng = np.random.default_rng([case["N"], case["S"], case["E"]])
    used = case["N"] - int(rng.integers(0, case["N"] // 16 + 1))
    share = rng.gamma(2.0, size=case["S"])
    return rng.multinomial(used, share / share.sum()).tolist()


_FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(e):
    """2^e in 32 bits for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _block_exponent(t):
    """The smallest e with absmax <= 6 * 2^e of each run of 32 values, in [-124, 125]."""
    amax = t.float().reshape(*t.shape[:-1], -1, 32).abs().amax(-1)
    m, p = torch.frexp(amax)  # amax = m 2^p, 6 = 0.75 * 2^3
    return (p - torch.where(m <= 0.75, 3, 2)).clamp(-124, 125)


def _nearest(a):
    """Index of the 4-bit magnitude nearest to a >= 0; ties to the even one."""
    i = (a > 0.25).to(torch.uint8)
    for edge, closed in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        i += (a >= edge) if closed else (a > edge)
    return i


def _plain_quant(t):
    """(bytes [..., cols / 2], even column in the low half; scale bytes [..., cols / 32])."""
    e = _block_exponent(t)
    v = t.float().reshape(*t.shape[:-1], -1, 32) * _pow2(-e).unsqueeze(-1)
    n = _nearest(v.abs()) | ((v < 0).to(torch.uint8) << 3)
    n = n.reshape(*t.shape[:-1], -1, 2)
    return n[..., 0] | (n[..., 1] << 4), (e + 127).to(torch.uint8)


def _plain_dequant(q, scale, dtype):
    pairs = torch.tensor([[(-1.0 if n & 8 else 1.0) * _FP4[n & 7] for n in (b & 15, b >> 4)] for b in range(256)],
                         dtype=torch.float32, device=q.device)
    v = pairs[q.int()].reshape(*scale.shape, 32)
    return (v * _pow2(scale.int() - 127).unsqueeze(-1)).reshape(*q.shape[:-1], -1).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def randn(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)

    s = {"case": case}
    if kind == "quant":
        s["t"] = randn(case["rows"], case["cols"], std=1.0 / math.sqrt(case["cols"]), dtype=_DT[case["dtype"]])
        return s
    if kind == "balance":
        N, E, K, S = case["N"], case["E"], case["K"], case["S"]
        s["logits"] = randn(N, E, dtype=torch.float32) + randn(E, std=0.5, dtype=torch.float32)
        s["idx"] = torch.topk(s["logits"], K, dim=-1).indices
        s["mask"] = None
        if case["mask"]:
            s["mask"] = torch.rand(N, device="cuda", generator=g) < 0.85
            # padding rows hold what a layer leaves there
            s["logits"][~s["mask"]] = float("nan")
        lengths = torch.tensor(_seq_lengths(case))
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).to("cuda")
        s["grad_balance"] = randn(1, dtype=torch.float32).reshape(()).abs() + 0.5
        s["grad_z"] = randn(1, dtype=torch.float32).reshape(()).abs() + 0.5
        return s
    R, H, F, E = case["R"], case["H"], case["F"], case["E"]
    order = torch.randperm(E, generator=torch.Generator().manual_seed(seed))
    counts = torch.tensor(_counts(case))[order]
    s["counts"] = counts.tolist()
    s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).to("cuda")
    s["wq"], s["wscale"] = [], []
    for rows, cols in ((F, H), (F, H), (H, F)):
        q = torch.empty(E, rows, cols // 2, dtype=torch.uint8, device="cuda")
        sc = torch.empty(E, rows, cols // 32, dtype=torch.uint8, device="cuda")
        for e in range(E):
            q[e], sc[e] = _plain_quant(randn(rows, cols, std=1.0 / math.sqrt(cols)))
        s["wq"].append(q)
        s["wscale"].append(sc)
    if kind == "experts":
        s["x"] = randn(R, H)
    else:
        s["dy"], s["hgu"] = randn(R, H), randn(R, 2 * F)
    return s


# ---- one pass ----


def _padded(t, s):
    """Rows [R, C] grouped by expert as [E, most rows of one, C] in 32 bits, zeros behind each expert's rows, and where
    each row went."""
    counts = torch.diff(s["offsets"]).long()
    most = max(s["counts"])
    row = torch.arange(t.shape[0], device=t.device)
    e = torch.bucketize(row, s["offsets"][1:].long(), right=True)
    at = e * most + (row - s["offsets"].long()[e])
    out = torch.zeros(len(counts) * most, t.shape[1], device=t.device)
    out[at] = t.float()
    return out.reshape(len(counts), most, -1), at


def _rows(t, at):
    return t.reshape(-1, t.shape[-1])[at]


def _plain_experts(s):
    wg, wu, wd = (_plain_dequant(q, sc, torch.float32) for q, sc in zip(s["wq"], s["wscale"]))
    x, at = _padded(s["x"], s)
    g, u = torch.bmm(x, wg.transpose(1, 2)), torch.bmm(x, wu.transpose(1, 2))
    y = torch.bmm(g / (1 + torch.exp(-g)) * u, wd.transpose(1, 2))
    out = {"y": _rows(y, at).to(torch.bfloat16)}
    if s["case"]["keep"]:
        out["hgu"] = torch.cat([_rows(g, at), _rows(u, at)], 1).to(torch.bfloat16)
    return out


def _plain_experts_bwd(s):
    wg, wu, wd = (_plain_dequant(q, sc, torch.float32) for q, sc in zip(s["wq"], s["wscale"]))
    dy, at = _padded(s["dy"], s)
    h, _ = _padded(s["hgu"], s)
    g, u = h.chunk(2, -1)
    da = torch.bmm(dy, wd)
    sig = 1 / (1 + torch.exp(-g))
    dx = torch.bmm(da * u * sig * (1 + g * (1 - sig)), wg) + torch.bmm(da * g * sig, wu)
    return {"dx": _rows(dx, at).to(torch.bfloat16)}


def _plain_balance(s):
    case, logits, idx = s["case"], s["logits"], s["idx"]
    N, E, K, S = case["N"], case["E"], case["K"], case["S"]
    seq = torch.bucketize(torch.arange(N, device=logits.device), s["offsets"][1:], right=True)
    valid = seq < S
    if s["mask"] is not None:
        valid = valid & s["mask"]
    seq = seq.clamp(max=S - 1)
    lg = torch.where(valid.unsqueeze(1), logits, 0.0)
    m = lg.amax(1, keepdim=True)
    ex = torch.exp(lg - m)
    tot = ex.sum(1, keepdim=True)
    p, lse = ex / tot, (m + torch.log(tot)).squeeze(1)
    v = valid.unsqueeze(1)

    def by_sequence(t):  # sums of consecutive rows as differences of the running sum, 64 bits wide
        run = torch.nn.functional.pad(t.reshape(N, -1).T.contiguous().cumsum(1), (1, 0))
        return (run[:, s["offsets"][1:]] - run[:, s["offsets"][:-1]]).T.reshape(S, *t.shape[1:])

    n = by_sequence(valid.long())
    hits = torch.zeros(N, E, dtype=torch.int64, device=logits.device).scatter_(1, idx, 1)
    cnt = by_sequence(hits * v)
    P = by_sequence(torch.where(v, p, 0.0).double())
    nd = n.clamp(min=1).double().unsqueeze(1)
    P = P / nd
    f = cnt.double() * (E / K) / nd
    used, total = (n > 0).sum(), n.sum()
    balance = _BALANCE * (f * P).sum() / used.clamp(min=1)
    z = _Z * torch.where(valid, lse.double() ** 2, 0.0).sum() / total.clamp(min=1)
    ft = f.float()[seq]
    cb = s["grad_balance"] * _BALANCE / used.clamp(min=1) / n.clamp(min=1)[seq].float()
    cz = s["grad_z"] * _Z * 2 / total.clamp(min=1)
    d = p * (cb.unsqueeze(1) * (ft - (p * ft).sum(1, keepdim=True)) + cz * lse.unsqueeze(1))
    return {"balance": balance.float(), "z": z.float(), "counts": cnt, "tokens": torch.cat([n, total.view(1), used.view(1)]),
            "mean_prob": P.float(), "dlogits": torch.where(v, d, 0.0)}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from moe_mi355 import ops

        if kind == "quant":
            return {"values": ops.dequant_mxfp4(*ops.quant_mxfp4(s["t"]), dtype=s["t"].dtype)}
        if kind == "experts":
            hgu, y = ops.swiglu_forward_mxfp4(s["x"], s["wq"], s["wscale"], s["offsets"], keep_preact=case["keep"])
            return {"y": y, "hgu": hgu} if case["keep"] else {"y": y}
        if kind == "experts_bwd":
            return {"dx": ops.swiglu_backward_mxfp4(s["dy"], s["hgu"], s["wq"], s["wscale"], s["offsets"])}
        balance, z, counts, tokens, mean_prob = ops.balance_loss_forward(
            s["logits"], s["idx"], s["offsets"], s["mask"], balance_coef=_BALANCE, z_coef=_Z)
        d = ops.balance_loss_backward(s["logits"], counts, tokens, case["K"], s["offsets"], s["mask"],
                                      s["grad_balance"], s["grad_z"], balance_coef=_BALANCE, z_coef=_Z)
        return {"balance": balance, "z": z, "counts": counts, "tokens": tokens, "mean_prob": mean_prob, "dlogits": d}
    if kind == "quant":
        return {"values": _plain_dequant(*_plain_quant(s["t"]), s["t"].dtype)}
    if kind == "experts":
        return _plain_experts(s)
    if kind == "experts_bwd":
        return _plain_experts_bwd(s)
    return _plain_balance(s)


# ---- what a pass cannot do without ----


def work(case):
    kind = case["kind"]
    if kind == "quant":  # read, write the 4-bit form, read it, write the values
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * (2 if case["dtype"] == "bf16" else 4) + 2 * (0.5 + 1 / 32)), "flops": 2 * n}
    if kind == "balance":
        N, E, K, S = case["N"], case["E"], case["K"], case["S"]
        # logits for the loss and for its gradient, the ids, the gradient; counts and means of each sequence
        return {"bytes": 12 * N * E + 8 * N * K + 20 * S * E + 16 * S + (2 * N if case["mask"] else 0), "flops": 16 * N * E}
    R, H, F = case["R"], case["H"], case["F"]
    live = sum(c > 0 for c in _counts(case))
    weights = live * 3 * F * H * (0.5 + 1 / 32)
    rows = R * 2 * (2 * H + (2 * F if kind == "experts_bwd" or case["keep"] else 0))
    return {"bytes": weights + rows, "flops": 6 * R * F * H}


# ---- the same in 64 bits ----


def _exact_values(q, scale):
    """The values of a 4-bit matrix, from the bits: sign, two of exponent, one of mantissa."""
    n = torch.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1).to(torch.int32)
    ex, man = (n >> 1) & 3, (n & 1).double()
    v = torch.where(ex == 0, man * 0.5, torch.ldexp(1 + 0.5 * man, ex - 1)) * (1 - 2 * (n >> 3).double())
    return torch.ldexp(v, (scale.to(torch.int32) - 127).repeat_interleave(32, -1))


def _exact_quant(t):
    v = t.double().reshape(t.shape[0], -1, 32)
    amax = v.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((amax / 6).clamp(min=2.0 ** -140))).clamp(-124, 125)
    e = torch.where(amax > 6 * torch.exp2(e), e + 1, torch.where(amax <= 3 * torch.exp2(e), e - 1, e)).clamp(-124, 125)
    a = v / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=1.0))) - 1)  # 1/2 below 2, then 1, 2
    a = (torch.round(a / step) * step).clamp(-6, 6)  # torch.round takes ties to even
    return (a * torch.exp2(e)).reshape(t.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return {"values": torch.cat([_exact_quant(t) for t in s["t"].split(8192)])}
    if kind == "balance":
        N, E, K, S = case["N"], case["E"], case["K"], case["S"]
        lengths = torch.diff(s["offsets"]).cpu()
        of = torch.repeat_interleave(torch.arange(S), lengths)
        ok = torch.zeros(N, dtype=torch.bool)
        ok[:len(of)] = True
        if s["mask"] is not None:
            ok &= s["mask"].cpu()
        at = ok.nonzero().squeeze(1)
        of = of[at]
        lg = s["logits"].cpu().double()[at].requires_grad_(True)
        n = torch.bincount(of, minlength=S)
        cnt = torch.bincount((of.unsqueeze(1) * E + s["idx"].cpu()[at]).reshape(-1), minlength=S * E).reshape(S, E)
        nd = n.clamp(min=1).unsqueeze(1).double()
        P = torch.zeros(S, E, dtype=torch.float64).index_add(0, of, torch.softmax(lg, -1)) / nd
        used, total = max(1, int((n > 0).sum())), max(1, len(at))
        balance = _BALANCE / used * (E / K * cnt / nd * P).sum()
        z = _Z / total * (torch.logsumexp(lg, -1) ** 2).sum()
        g, = torch.autograd.grad(s["grad_balance"].cpu().double() * balance + s["grad_z"].cpu().double() * z, lg)
        d = torch.zeros(N, E, dtype=torch.float64)
        d[at] = g
        out = {"balance": balance.detach(), "z": z.detach(), "counts": cnt,
               "tokens": torch.cat([n, n.sum().view(1), (n > 0).sum().view(1)]), "mean_prob": P.detach(), "dlogits": d}
        return {k: t.to("cuda") for k, t in out.items()}
    F = case["F"]
    parts = {}
    bounds = s["offsets"].tolist()
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo == hi:
            continue
        wg, wu, wd = (_exact_values(q[e], sc[e]) for q, sc in zip(s["wq"], s["wscale"]))
        if kind == "experts":
            x = s["x"][lo:hi].double()
            g, u = x @ wg.T, x @ wu.T
            parts.setdefault("y", []).append((g * torch.sigmoid(g) * u) @ wd.T)
            if case["keep"]:
                parts.setdefault("hgu", []).append(torch.cat([g, u], 1))
        else:
            g, u = (t.double().requires_grad_(True) for t in (s["hgu"][lo:hi, :F], s["hgu"][lo:hi, F:]))
            dg, du = torch.autograd.grad(torch.nn.functional.silu(g) * u, (g, u), s["dy"][lo:hi].double() @ wd)
            parts.setdefault("dx", []).append(dg @ wg + du @ wu)
    return {k: torch.cat(v) for k, v in parts.items()}
