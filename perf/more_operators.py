"""Operators of a block that is trained in bf16 / fp32 and served in 8-bit integers: the norm with the residual's addition, and
matrix products on int8 rows and weights with a scale for each token and output channel.

Kinds of case:

norm_train  h = x + residual and its RMSNorm, and the gradients of both (they share one) and of the weight
norm_quant  the same for serving: the normalised rows in 8 bits with a scale each (int8 or e4m3), read back as values
product     rows quantized to int8, times an int8 weight matrix, or times each row group's own
experts     tokens quantized to int8, through the SwiGLU experts that they are routed to, on int8 weights

The plain forms work in 32 bits (64 for long sums) and round once at the end.  The experts' activations are a bf16 tensor by
definition, as in the bf16 layer that is quantized: they are rounded there too before they become int8.  ``exact`` works in
64 bits.
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
_EPS = 1e-5  # RMSNorm's default


def listed():
    return [
        # training in fp32, a small layer
        {"name": "norm_train_small", "kind": "norm_train", "dtype": "f32", "N": 4096, "H": 512},
        # training in bf16: a batch of a wide layer
        {"name": "norm_train_wide", "kind": "norm_train", "dtype": "bf16", "N": 16384, "H": 4096},
        # one decoded token between two blocks: latency counts
        {"name": "norm_quant_one_token", "kind": "norm_quant", "dtype": "bf16", "N": 1, "H": 4096, "residual": True,
         "format": "int8", "keep": False},
        # a long prompt; the router reads the normalised rows in bf16, the experts in 8 bits
        {"name": "norm_quant_prompt", "kind": "norm_quant", "dtype": "bf16", "N": 65536, "H": 2048, "residual": True,
         "format": "e4m3", "keep": True},
        # a projection of a decode step of 16 sequences: the weights are all there is to read
        {"name": "product_decode", "kind": "product", "dtype": "bf16", "R": 16, "K": 4096, "N": 4096, "E": 0, "skew": 0.0},
        # the same of a prompt, an odd number of rows
        {"name": "product_prompt", "kind": "product", "dtype": "bf16", "R": 8190, "K": 4096, "N": 14336, "E": 0, "skew": 0.0},
        # a projection of many small experts, unevenly filled, fp32 rows
        {"name": "product_grouped", "kind": "product", "dtype": "f32", "R": 24570, "K": 2048, "N": 768, "E": 64, "skew": 1.1},
        # one decoded token through its two experts
        {"name": "experts_one_token", "kind": "experts", "T": 1, "K": 2, "H": 4096, "F": 14336, "E": 8, "skew": 0.0},
        # a decode step of 64 sequences, every expert in use
        {"name": "experts_decode", "kind": "experts", "T": 64, "K": 2, "H": 4096, "F": 14336, "E": 8, "skew": 0.0},
        # a decode step over many small experts, 8 each, unevenly routed
        {"name": "experts_decode_small", "kind": "experts", "T": 64, "K": 8, "H": 2048, "F": 768, "E": 128, "skew": 1.1},
        # a chunk of a prompt beside running decodes: rows enough that neither weights nor products bound it alone
        {"name": "experts_chunk", "kind": "experts", "T": 501, "K": 2, "H": 4096, "F": 14336, "E": 8, "skew": 0.0},
        # a long prompt
        {"name": "experts_prompt", "kind": "experts", "T": 8192, "K": 2, "H": 4096, "F": 14336, "E": 8, "skew": 0.0},
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm_train", "norm_quant", "product", "product", "experts", "experts"])
    if kind.startswith("norm"):
        H = 16 * _logint(rng, 1, 512)
        c = {"kind": kind, "dtype": rng.choice(["bf16", "f32"]), "N": _logint(rng, 1, min(65536, 16384 * 4096 // H)), "H": H}
        if kind == "norm_quant":
            c.update(residual=rng.random() < 0.5, format=rng.choice(["int8", "e4m3"]), keep=rng.random() < 0.5)
        return c
    while True:
        if kind == "product":
            c = {"kind": kind, "dtype": rng.choice(["bf16", "f32"]), "R": _logint(rng, 1, 32768), "K": 16 * _logint(rng, 2, 896),
                 "N": 8 * _logint(rng, 2, 1792), "E": rng.choice([0, _logint(rng, 2, 128)]), "skew": rng.choice([0.0, 1.1])}
            E = max(1, c["E"])
            room = E * max(_product_counts(c)) * (c["K"] + c["N"])
            if c["R"] * c["K"] * c["N"] <= 8190 * 4096 * 14336 and E * c["K"] * c["N"] <= 1 << 29 and room <= 1 << 30:
                return c
        else:
            E = _logint(rng, 1, 128)
            c = {"kind": kind, "T": _logint(rng, 1, 8192), "K": rng.randint(1, min(8, E)), "H": 16 * _logint(rng, 8, 256),
                 "F": 32 * _logint(rng, 4, 448), "E": E, "skew": rng.choice([0.0, 1.1])}
            room = E * int(np.bincount(_choices(c).reshape(-1), minlength=E).max()) * (2 * c["F"] + c["H"])
            if (E * c["F"] * c["H"] <= 8 * 14336 * 4096 and c["T"] * c["K"] * c["F"] * c["H"] <= 16384 * 14336 * 4096
                    and room <= 1 << 30):
                return c


# ---- inputs ----


def _product_counts(case):
    """Rows of each group, the largest share first where they are uneven (Zipf); one group without experts."""
    if case["E"] == 0:
        return [case["R"]]
    share = (1.0 + np.arange(case["E"])) ** -case["skew"]
    rng = np.random.default_rng([case["R"], case["E"], case["K"], case["N"]])
    return rng.multinomial(case["R"], share / share.sum()).tolist()


def _choices(case):
    """Each token's K experts: the largest of random logits, with a Zipf bias where the routing is skewed."""
    rng = np.random.default_rng([case["T"], case["K"], case["E"], case["H"], case["F"]])
    logits = rng.normal(size=(case["T"], case["E"])) - case["skew"] * np.log1p(np.arange(case["E"]))
    return np.argsort(-logits, axis=1)[:, :case["K"]]


_TINY = 2.0 ** -100


def _plain_quant(v):
    """Rows of 32-bit values in int8, with their scales; a row that holds an infinity or a NaN stands for NaNs.  The quotient is
    taken in 64 bits: in 32 a value next to the border between two whole numbers (half of the row's largest is on it) may fall
    on either side."""
    a = v.abs().amax(-1, keepdim=True).clamp(min=_TINY)
    ok = torch.isfinite(v).all(-1, keepdim=True)
    q = torch.where(ok, torch.round(v.double() * 127.0 / a.double()), 0.0).to(torch.int8)
    return q, torch.where(ok, a / 127.0, float("nan")).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def randn(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)

    def weights(E, rows, cols):
        q = torch.empty(E, rows, cols, dtype=torch.int8, device="cuda")
        s = torch.empty(E, rows, device="cuda")
        for e in range(E):
            q[e], s[e] = _plain_quant(randn(rows, cols, std=1.0 / math.sqrt(cols), dtype=torch.float32))
        return q, s

    s = {"case": case}
    if kind.startswith("norm"):
        N, H, dt = case["N"], case["H"], _DT[case["dtype"]]
        s["x"] = randn(N, H, dtype=dt)
        s["weight"] = 1.0 + randn(H, std=0.1, dtype=torch.float32)
        if kind == "norm_train" or case["residual"]:
            s["residual"] = randn(N, H, std=2.0, dtype=dt)
        if kind == "norm_train":
            s["dxn"], s["dh"] = randn(N, H, dtype=dt), randn(N, H, dtype=dt)
        return s
    if kind == "product":
        order = torch.randperm(max(1, case["E"]), generator=torch.Generator().manual_seed(seed))
        counts = torch.tensor(_product_counts(case))[order]
        s["x"] = randn(case["R"], case["K"], dtype=_DT[case["dtype"]])
        s["wq"], s["wscale"] = weights(max(1, case["E"]), case["N"], case["K"])
        s["offsets"] = None
        if case["E"] == 0:
            s["wq"], s["wscale"] = s["wq"][0], s["wscale"][0]
    else:
        # the plan of the routing that the program made before: rows grouped by expert, each with its token's slot
        T, K, H, F, E = case["T"], case["K"], case["H"], case["F"], case["E"]
        cpu = torch.Generator().manual_seed(seed)
        idx = torch.randperm(E, generator=cpu)[torch.from_numpy(_choices(case))][torch.randperm(T, generator=cpu)].reshape(-1)
        counts = torch.bincount(idx, minlength=E)
        s["row_slot"] = torch.argsort(idx, stable=True).to(torch.int32).to("cuda")
        s["x"] = randn(T, H)
        made = [weights(E, F, H), weights(E, F, H), weights(E, H, F)]
        s["wq"], s["wscale"] = [q for q, _ in made], [t for _, t in made]
    s["counts"] = counts.tolist()
    if kind == "experts" or case["E"]:
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).to("cuda")
    return s


# ---- one pass ----


def _plain_norm(s):
    """(h in the inputs' type, 1 / rms in 32 bits, the normalised rows in 32 bits)."""
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype) if "residual" in s else s["x"]
    v = h.float()
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
    return h, r, v * r * s["weight"]


def _plain_norm_train(s):
    h, r, xn = _plain_norm(s)
    dt = h.dtype
    xhat, u = h.float() * r, s["dxn"].float()
    g = u * s["weight"]
    d = s["dh"].float() + r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    return {"h": h, "xn": xn.to(dt), "d": d.to(dt), "dweight": (u * xhat).sum(0, dtype=torch.float64).float()}


def _plain_norm_quant(s):
    case = s["case"]
    h, _, xn = _plain_norm(s)
    if case["format"] == "int8":
        q, scale = _plain_quant(xn)
        values = q.float() * scale.unsqueeze(-1)
    else:
        a = xn.abs().amax(-1, keepdim=True)
        tiny = a < 2.0 ** -118
        scale = torch.where(tiny, 1.0, a / 448.0)
        q = (xn * torch.where(tiny, 1.0, torch.full_like(a, 448.0) / a)).to(torch.float8_e4m3fn)
        values, scale = q.float() * scale, scale.squeeze(-1)
    out = {"scale": scale, "values": values.to(torch.bfloat16)}
    if case["residual"]:
        out["h"] = h
    if case["keep"]:
        out["xn"] = xn.to(s["x"].dtype)
    return out


def _padded(t, s):
    """Rows [R, C] grouped by expert as [E, most rows of one, C], zeros behind each expert's rows, and where each row went."""
    counts = torch.diff(s["offsets"]).long()
    most = max(s["counts"])
    row = torch.arange(t.shape[0], device=t.device)
    e = torch.bucketize(row, s["offsets"][1:].long(), right=True)
    at = e * most + (row - s["offsets"].long()[e])
    out = torch.zeros(len(counts) * most, t.shape[1], device=t.device)
    out[at] = t.float()
    return out.reshape(len(counts), most, -1), at


def _plain_product(q, scale, wq, wscale, s):
    """Scaled products of int8 rows with int8 weights, in 32 bits (each partial sum is a whole number)."""
    if s["offsets"] is None:
        return (q.float() @ wq.float().T) * scale.unsqueeze(1) * wscale
    x, at = _padded(q, s)
    y = torch.bmm(x, wq.float().transpose(1, 2).contiguous()) * wscale.unsqueeze(1)
    return y.reshape(-1, y.shape[-1])[at] * scale.unsqueeze(1)


def _plain_experts(s):
    rows = s["row_slot"].long() // s["case"]["K"]
    q, scale = _plain_quant(s["x"].float())
    q, scale = q[rows], scale[rows]
    g = _plain_product(q, scale, s["wq"][0], s["wscale"][0], s)
    u = _plain_product(q, scale, s["wq"][1], s["wscale"][1], s)
    act = (g / (1 + torch.exp(-g)) * u).to(torch.bfloat16)
    return {"y": _plain_product(*_plain_quant(act.float()), s["wq"][2], s["wscale"][2], s).to(torch.bfloat16)}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from moe_mi355 import ops

        if kind == "norm_train":
            xn, h, rstd = ops.rmsnorm_residual_forward(s["x"], s["residual"], s["weight"], _EPS)
            d, dweight = ops.rmsnorm_residual_backward(h, s["weight"], rstd, s["dxn"], s["dh"])
            return {"h": h, "xn": xn, "d": d, "dweight": dweight}
        if kind == "norm_quant":
            q, scale, xn, h = ops.rmsnorm_quant(s["x"], s["weight"], _EPS, residual=s.get("residual"), fmt=case["format"],
                                                keep_norm=case["keep"])
            out = {"scale": scale, "values": ops.dequant_rows(q, scale, torch.bfloat16)}
            if case["residual"]:
                out["h"] = h
            if case["keep"]:
                out["xn"] = xn
            return out
        if kind == "product":
            q, scale = ops.quant_rows_int8(s["x"])
            return {"y": ops.matmul_int8(q, scale, s["wq"], s["wscale"], offsets=s["offsets"], out_dtype=s["x"].dtype)}
        q, scale = ops.quant_rows_int8(s["x"])
        return {"y": ops.swiglu_forward_int8(q, scale, s["wq"], s["wscale"], s["offsets"], row_slot=s["row_slot"],
                                             top_k=case["K"])}
    if kind == "norm_train":
        return _plain_norm_train(s)
    if kind == "norm_quant":
        return _plain_norm_quant(s)
    if kind == "product":
        q, scale = _plain_quant(s["x"].float())
        return {"y": _plain_product(q, scale, s["wq"], s["wscale"], s).to(s["x"].dtype)}
    return _plain_experts(s)


# ---- what a pass cannot do without ----


def work(case):
    kind = case["kind"]
    if kind.startswith("norm"):
        n, size = case["N"] * case["H"], 2 if case["dtype"] == "bf16" else 4
        if kind == "norm_train":  # x, residual, dxn, dh, h read; h, xn, d written
            return {"bytes": 8 * n * size + 12 * case["H"], "flops": 20 * n}
        # x (residual) read; bytes (h, xn) written; the bytes read again as bf16 values
        tensors = 1 + 2 * case["residual"] + case["keep"]
        return {"bytes": n * (tensors * size + 1 + 1 + 2) + 8 * case["N"] + 4 * case["H"], "flops": 10 * n}
    if kind == "product":
        R, K, N = case["R"], case["K"], case["N"]
        size = 2 if case["dtype"] == "bf16" else 4
        live = sum(c > 0 for c in _product_counts(case))
        return {"bytes": R * K * size + live * (N * K + 4 * N) + R * N * size, "flops": 2 * R * K * N}
    T, K, H, F = case["T"], case["K"], case["H"], case["F"]
    live = len(np.unique(_choices(case)))
    return {"bytes": 2 * T * H + live * (3 * F * H + 4 * (2 * F + H)) + 2 * T * K * H, "flops": 6 * T * K * F * H}


# ---- the same in 64 bits ----


def _exact_quant(v):
    """(whole numbers, scales) of rows of 64-bit values."""
    m = torch.maximum(v.max(-1, keepdim=True).values, -v.min(-1, keepdim=True).values).clamp(min=_TINY)
    return torch.round(127 * v / m), (m / 127).squeeze(-1)


def _exact_e4m3(v):
    """Nearest value with three bits behind the leading one, an exponent of at least -6 and at most 448; ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("norm"):
        h = s["x"]
        if "residual" in s:
            h = (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
        v, w = h.double(), s["weight"].double()
        rms = (v.square().sum(-1, keepdim=True) / case["H"] + _EPS).sqrt()
        xn = v / rms * w
        if kind == "norm_train":
            u = s["dxn"].double()
            dot = (u * w * v).sum(-1, keepdim=True) / case["H"]
            return {"h": h.double(), "xn": xn, "d": s["dh"].double() + u * w / rms - v * dot / rms ** 3,
                    "dweight": (u * v / rms).sum(0)}
        if case["format"] == "int8":
            q, scale = _exact_quant(xn)
        else:
            scale = xn.abs().amax(-1) / 448
            scale = torch.where(scale < 2.0 ** -118 / 448, torch.ones_like(scale), scale)
            q = _exact_e4m3(xn / scale.unsqueeze(-1))
        out = {"scale": scale, "values": q * scale.unsqueeze(-1)}
        if case["residual"]:
            out["h"] = h.double()
        if case["keep"]:
            out["xn"] = xn
        return out
    if kind == "product":
        q, scale = _exact_quant(s["x"].double())
        bounds = [0, case["R"]] if s["offsets"] is None else s["offsets"].tolist()
        wq, ws = s["wq"].reshape(-1, *s["wq"].shape[-2:]), s["wscale"].reshape(-1, s["wscale"].shape[-1])
        y = [(q[a:b] @ wq[e].double().T) * scale[a:b, None] * ws[e].double() for e, (a, b) in enumerate(zip(bounds, bounds[1:]))]
        return {"y": torch.cat(y)}
    q, scale = _exact_quant(s["x"].double())
    token = torch.div(s["row_slot"].long(), case["K"], rounding_mode="floor")
    parts, bounds = [], s["offsets"].tolist()
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if a == b:
            continue
        gate, up, down = (w[e].double() * t[e].double().unsqueeze(1) for w, t in zip(s["wq"], s["wscale"]))
        x = q[token[a:b]] * scale[token[a:b], None]
        g = x @ gate.T
        act = (g * torch.sigmoid(g) * (x @ up.T)).to(torch.bfloat16).double()
        aq, sa = _exact_quant(act)
        parts.append((aq @ down.T) * sa.unsqueeze(1))
    return {"y": torch.cat(parts)}
