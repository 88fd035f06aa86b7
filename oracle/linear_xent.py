"""Cross entropy of a linear head from its definition, in 64 bits, on its
inputs' device, with what roundings can change.

`u` is half a step of the type that dz and the gradients are rounded to,
`least` what the smallest of its values can be off by.  Sums of n products by
32-deep matrix instructions pass at most n / 32 + 32 roundings of 2^-23."""

import torch


def _depth(n):
    return (n / 32 + 32) * 2.0**-23


def linear_xent(h, w, labels, ignore_index=-100, dloss=None, u=0.0, least=0.0, floor=0.0):
    """{"loss", "dh", "dw"} of h [rows, H], w [V, H], labels [rows] (clamped to
    the vocabulary), gradients where `dloss` is given, and under "bound_..." how
    far roundings can put each.  floor: the smallest dz that a rounding keeps,
    relative to dloss."""
    h, w = h.double(), w.double()
    V, H = w.shape
    on = labels != ignore_index
    hz = torch.where(on[:, None], h, 0.0)
    t = labels.clamp(0, V - 1)
    z = hz @ w.T
    ez = _depth(H) * (hz.abs() @ w.abs().T)
    top = z.amax(1, keepdim=True)
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    spread = (p * (top - z)).sum(1)
    pick = lambda x: x.gather(1, t[:, None])[:, 0]  # noqa: E731
    r = {"loss": torch.where(on, -pick(logp), 0.0)}
    # the sum of exponentials: 120 additions, each term off by its exponent's rounding; z once for the row and once
    # for its label
    el = 120 * 2.0**-24 + (1 + spread) * 2.0**-22 + (p * ez).sum(1) + top[:, 0].abs() * 2.0**-23
    r["bound_loss"] = torch.where(on, el + pick(ez) + pick(logp).abs() * 2.0**-22 + pick(z).abs() * 2.0**-23, 0.0)
    if dloss is None:
        return r
    g = torch.where(on, dloss.double(), 0.0)[:, None]
    dz = p.clone()
    dz.scatter_add_(1, t[:, None], torch.full_like(dz[:, :1], -1.0))
    edz = p * (ez + el[:, None] + (1 + logp.abs()) * 2.0**-21) + (u + 2.0**-22) * dz.abs() + floor
    dz, edz = dz * g, edz * g.abs()
    r["dh"], r["dw"] = dz @ w, dz.T @ hz
    deep = _depth(V) + 64 * 2.0**-23
    r["bound_dh"] = (edz + deep * dz.abs()) @ w.abs() + 1.001 * u * r["dh"].abs() + least
    r["bound_dw"] = (edz + _depth(h.shape[0]) * dz.abs()).T @ hz.abs() + 1.001 * u * r["dw"].abs() + least
    return r
