"""CPU restatement of the balance loss of sequences and the z-loss over valid tokens -- TEST INFRASTRUCTURE ONLY.

The reference has no load-balance loss and a detached z-loss (moe-engine/pkg/kernels/moe_router.py L:603-612).  In float64,
sequence by sequence:

    balance = balance_coef * mean over sequences with valid tokens of sum_e (E c_e / (K n)) mean_t p[t, e]
    z       = z_coef * mean over valid tokens of logsumexp(logits_t)^2

Pinning (``tests/test_oracle_balance.py``): against ``oracle.router``'s whole-batch losses for one sequence without a mask,
and the gradient against central differences.
"""

from __future__ import annotations

from typing import Optional

import torch


def balance(logits: torch.Tensor, idx: torch.Tensor, offsets: Optional[torch.Tensor] = None,
            mask: Optional[torch.Tensor] = None, balance_coef: float = 1.0, z_coef: float = 0.0,
            grad_balance: float = 1.0, grad_z: float = 1.0) -> dict:
    """balance, z, counts [S, E], tokens [S + 2], mean_prob [S, E] and dlogits [N, E] (the gradient of
    grad_balance * balance + grad_z * z), the counts taken as constants."""
    N, E = logits.shape
    K = idx.shape[1]
    bounds = [0, N] if offsets is None else [int(v) for v in offsets]
    S = len(bounds) - 1
    ok = torch.ones(N, dtype=torch.bool) if mask is None else mask.reshape(-1).clone()
    counts = torch.zeros(S, E, dtype=torch.int64)
    mean_prob = torch.zeros(S, E, dtype=torch.float64)
    tokens = torch.zeros(S + 2, dtype=torch.int64)
    frac = torch.zeros(S, E, dtype=torch.float64)
    rows = []
    for s in range(S):
        t = torch.arange(bounds[s], bounds[s + 1])
        t = t[ok[t]]
        rows.append(t)
        n = len(t)
        tokens[s] = n
        if n == 0:
            continue
        choices = idx[t].reshape(-1)
        counts[s] = torch.bincount(choices[(choices >= 0) & (choices < E)], minlength=E)
        mean_prob[s] = torch.softmax(logits[t].double(), -1).mean(0)
        frac[s] = E * counts[s].double() / (K * n)
    n, used = int(tokens.sum()), int((tokens[:S] > 0).sum())
    tokens[S], tokens[S + 1] = n, used
    d = torch.zeros(N, E, dtype=torch.float64)
    zsum = 0.0
    for s, t in enumerate(rows):
        if len(t) == 0:
            continue
        lg = logits[t].double()
        p, lse = torch.softmax(lg, -1), torch.logsumexp(lg, -1, keepdim=True)
        zsum += float((lse ** 2).sum())
        d[t] = (grad_balance * balance_coef / (used * len(t)) * p * (frac[s] - (p * frac[s]).sum(-1, keepdim=True))
                + grad_z * z_coef * 2.0 / n * lse * p)
    loss = balance_coef * float((frac * mean_prob).sum()) / max(used, 1)
    return {"balance": torch.tensor(loss, dtype=torch.float64), "z": torch.tensor(z_coef * zsum / max(n, 1), dtype=torch.float64),
            "counts": counts, "tokens": tokens, "mean_prob": mean_prob, "dlogits": d}
