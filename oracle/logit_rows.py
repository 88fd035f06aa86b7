"""Token log probabilities and distillation from a teacher's top logits, row by
row from their definitions, in the precision of their inputs (CPU)."""

import math

import torch


def _log_softmax(x):
    """(the maximum first: logits as far out as a type's lowest value absorb a
    row's log sum)"""
    d = x - x.max()
    return d - d.exp().sum().log()


def token_logprobs(z, tokens, top_k, ignore_index=-100, dlogprob=None, dentropy=None):
    """{"logprob", "entropy", "top", "ids", "logp", "spread"} of z [rows, V] and
    with upstream gradients also "dz"; "spread" is sum p |z - max|."""
    rows, V = z.shape
    r = {"logprob": z.new_zeros(rows), "entropy": z.new_zeros(rows), "spread": z.new_zeros(rows),
         "top": z.new_full((rows, top_k), -math.inf), "ids": torch.full((rows, top_k), -1, dtype=torch.int64),
         "logp": z.new_full((rows, V), -math.inf)}
    if dlogprob is not None or dentropy is not None:
        r["dz"] = torch.zeros_like(z)
    for i in range(rows):
        if tokens[i] == ignore_index:
            continue
        x, t = z[i], min(max(int(tokens[i]), 0), V - 1)
        # NaN first, then by value, equal ones by index
        order = sorted(range(V), key=lambda j: (0, 0, j) if x[j].isnan() else (1, -float(x[j]), j))[:top_k]
        r["ids"][i] = torch.tensor(order, dtype=torch.int64)
        if (x == -math.inf).all():
            r["logprob"][i] = -math.inf
            continue
        logp = _log_softmax(x)
        if x.isnan().any() or (x == math.inf).any():
            logp = torch.full_like(x, math.nan)
        r["logp"][i], p = logp, logp.exp()
        plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
        r["logprob"][i], r["entropy"][i], r["top"][i] = logp[t], -plogp.sum(), logp[order]
        r["spread"][i] = torch.where(p == 0, torch.zeros_like(p), p * (x.max() - x)).sum()
        if "dz" in r:
            g = float(dlogprob[i]) if dlogprob is not None else 0.0
            h = float(dentropy[i]) if dentropy is not None else 0.0
            if g or h:
                hit = torch.zeros_like(x)
                hit[t] = 1.0
                r["dz"][i] = g * (hit - p) - h * (plogp + p * r["entropy"][i])
    return r


def topk_distill(z, ids, teacher, temperature, dloss=None):
    """{"loss", "q" (the teacher's mass by id), "logp", "size" (sum q (1 + |log
    q| + |log p|))} of z [rows, V], and with `dloss` also "dz"."""
    rows, V = z.shape
    r = {"loss": z.new_zeros(rows), "size": z.new_zeros(rows), "q": torch.zeros_like(z),
         "logp": torch.full_like(z, -math.inf)}
    if dloss is not None:
        r["dz"] = torch.zeros_like(z)
    for i in range(rows):
        there = [j for j in range(ids.shape[1]) if 0 <= ids[i, j] < V and teacher[i, j] > -math.inf]
        if not there:
            continue
        q = torch.softmax(teacher[i, there] / temperature, 0)
        logp = _log_softmax(z[i] / temperature)
        if (z[i] == -math.inf).all():
            logp = torch.full_like(z[i], -math.inf)
        picked = logp[ids[i, there]]
        r["loss"][i] = temperature**2 * (q * (q.log() - picked)).sum()
        r["size"][i] = (q * (1 + q.log().abs() + picked.abs())).sum()
        r["logp"][i] = logp
        r["q"][i].index_add_(0, ids[i, there], q)
        if dloss is not None and not (z[i] == -math.inf).all():
            r["dz"][i] = float(dloss[i]) * temperature * (logp.exp() - r["q"][i])
    return r
