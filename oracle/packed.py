"""Causal attention over packed sequences with shared key and value heads, from
its definition, in the precision of its inputs (CPU).

Besides outputs and gradients it gives, per element, what one rounding of
relative size u in each place where a kernel rounds to 16 bits can change: P
and dS before the second products, and the stored results."""

import math

import torch


def packed_attention(q, k, v, lengths, scale=None, dout=None, u=0.0):
    """{"out", "lse"} of q [rows, n, hn] and k, v [rows, m, hn], with `dout`
    [rows, n, hn] also {"dq", "dk", "dv"}, and under "bound_..." the largest
    change that roundings of relative size u explain."""
    rows, n, hn = q.shape
    m = k.shape[1]
    scale = hn**-0.5 if scale is None else scale
    new = lambda *s: torch.zeros(*s, dtype=q.dtype)  # noqa: E731
    names = ["out", "bound_out"] + (["dq", "bound_dq"] if dout is not None else [])
    r = {name: new(rows, n, hn) for name in names}
    r["lse"] = torch.full((n, rows), -math.inf, dtype=q.dtype)
    if dout is not None:
        r |= {name: new(rows, m, hn) for name in ("dk", "dv", "bound_dk", "bound_dv")}
    a = 0
    for length in lengths:
        s = slice(a, a + length)
        a += length
        if not length:
            continue
        hidden = torch.ones(length, length, dtype=torch.bool).triu(1)
        for h in range(n):
            g = h // (n // m)
            score = (q[s, h] @ k[s, g].T * scale).masked_fill(hidden, -math.inf)
            r["lse"][h, s] = torch.logsumexp(score, 1)
            p = torch.softmax(score, 1)
            out = p @ v[s, g]
            r["out"][s, h] = out
            r["bound_out"][s, h] = u * (p @ v[s, g].abs() + out.abs())
            if dout is None:
                continue
            do = dout[s, h]
            ds = p * (do @ v[s, g].T - (do * out).sum(1, keepdim=True))
            # dS: its own rounding, and delta's from the rounded output
            eds = u * ds.abs() + p * (do.abs() * r["bound_out"][s, h]).sum(1, keepdim=True)
            r["dq"][s, h] = scale * (ds @ k[s, g])
            r["bound_dq"][s, h] = scale * (eds @ k[s, g].abs()) + u * r["dq"][s, h].abs()
            r["dk"][s, g] += scale * (ds.T @ q[s, h])
            r["bound_dk"][s, g] += scale * (eds.T @ q[s, h].abs())
            r["dv"][s, g] += p.T @ do
            r["bound_dv"][s, g] += u * (p.T @ do.abs())
    if dout is not None:
        for name in ("dk", "dv"):
            r["bound_" + name] += u * r[name].abs()
    return r
