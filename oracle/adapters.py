"""A projection with low-rank adapters of many tasks from its definition, in 64
bits, on its inputs' device, with what roundings can change.

`u` is half a step of the 16-bit type, `least` what its smallest values can be
off by, `floor` what the smallest of x A^T and dy B are off by, relative to the
largest.  Sums of n products by 32-deep matrix instructions pass at most n / 32 + 32
roundings of 2^-23 (and 16 more where the depth is split or chunks are joined)."""

import torch


def _depth(n):
    return (n / 32 + 48) * 2.0**-23


def adapter_linear(x, w, bias, lora_a, lora_b, of_row, scale, dy=None, u=0.0, least=0.0, floor=0.0):
    """{"y"} of x [rows, K], w [N, K], lora_a [adapters, r, K], lora_b [adapters,
    N, r] for rows of adapters of_row [rows] (-1: none) and scales [rows], with `dy`
    also {"dx", "da", "db"}, and under "bound_..." how far roundings can put each."""
    x, w, a, b, scale = (t.double() for t in (x, w, lora_a, lora_b, scale))
    rows, K = x.shape
    N, r = w.shape[0], a.shape[1]
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device=x.device)  # noqa: E731
    out = {"y": x @ w.T + (0.0 if bias is None else bias.double())}
    ey = _depth(K) * (x.abs() @ w.abs().T) + (0.0 if bias is None else 2.0**-23 * bias.double().abs())
    if dy is not None:
        dy = dy.double()
        out["dx"], edx = dy @ w, _depth(N) * (dy.abs() @ w.abs())
        out |= {"da": new(*a.shape), "db": new(*b.shape), "bound_da": new(*a.shape), "bound_db": new(*b.shape)}

    def narrow(rows, m, s):
        """s rows m^T as rounded to 16 bits, and its bound."""
        v = s * (rows @ m.T)
        size = torch.where(v.isfinite(), v.abs(), 0.0).max()
        return v, s.abs() * _depth(rows.shape[1]) * (rows.abs() @ m.abs().T) + (u + 2.0**-22) * v.abs() + floor * size

    for i in range(a.shape[0]):
        at = of_row == i
        if not at.any():
            continue
        s = scale[at, None]
        v, ev = narrow(x[at], a[i], s)
        out["y"][at] += v @ b[i].T
        ey[at] += (ev + _depth(r) * v.abs()) @ b[i].abs().T
        if dy is None:
            continue
        g, eg = narrow(dy[at], b[i].T, s)
        out["dx"][at] += g @ a[i]
        edx[at] += (eg + _depth(r) * g.abs()) @ a[i].abs()
        deep = _depth(int(at.sum()))
        out["da"][i] = g.T @ x[at]
        out["bound_da"][i] = (eg + deep * g.abs()).T @ x[at].abs()
        out["db"][i] = dy[at].T @ v
        out["bound_db"][i] = dy[at].abs().T @ (ev + deep * v.abs())
    out["bound_y"] = ey + 2.0**-22 * out["y"].abs()
    if dy is not None:
        out["bound_dx"] = edx
    for name in ("y", "dx", "da", "db"):
        if name in out:
            out["bound_" + name] += 1.001 * u * out[name].abs() + least
    return out
