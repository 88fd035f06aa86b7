"""The norm behind a block, its gate, the scaled residual and the norm before the
next block, from their definitions in 64 bits, with what the fp32 arithmetic and
the roundings to 16 bits can change.

`u` is half a step of the 16-bit type, `least` what its smallest values can be
off by.  A row's sum passes at most cols / 64 + 10 additions, a column's
rows / 256 + 40."""

import torch

STEP = 2.0**-23


def _norm(v, eps, rms, ev=0.0):
    """(vhat, inverse deviation, bound of vhat) of rows v in fp32, off by up to ev."""
    cols = v.shape[1]
    deep = (cols / 64 + 16) * STEP
    ev = torch.zeros_like(v) + ev
    mu = torch.zeros_like(v[:, :1]) if rms else v.mean(1, keepdim=True)
    inv = 1.0 / torch.sqrt(((v - mu) ** 2).mean(1, keepdim=True) + eps)
    hat = (v - mu) * inv
    off = torch.zeros_like(mu) if rms else inv * (deep * v.abs().mean(1, keepdim=True) + ev.mean(1, keepdim=True))
    # (the deviation's own change, relative to it: mean of |vhat| ev, over it)
    return hat, inv, off + inv * ev + hat.abs() * (deep + inv * (hat.abs() * ev).mean(1, keepdim=True))


def _back(g, eg, hat, ehat, inv, rms, einv=0.0):
    """(gradient of v, its bound) from that of vhat (g, off by up to eg); einv: what
    inv is off by, relative to it, beyond its rounding."""
    deep = (g.shape[1] / 64 + 16) * STEP
    mean = lambda x: x.mean(1, keepdim=True)  # noqa: E731
    s1, s2 = (torch.zeros_like(inv) if rms else mean(g)), mean(g * hat)
    e1 = torch.zeros_like(inv) if rms else mean(eg) + deep * mean(g.abs())
    e2 = mean(eg * hat.abs() + g.abs() * ehat) + deep * mean((g * hat).abs())
    out = inv * (g - s1 - hat * s2)
    size = g.abs() + s1.abs() + (hat * s2).abs()
    return out, inv * (eg + e1 + hat.abs() * e2 + ehat * s2.abs() + (deep + einv) * size)


def _stream(x, residual, pg, pb, gate, scale, eps, rms):
    """h in fp32 and its bound; xhat, its inverse deviation and its bound."""
    hat, inv, ehat = _norm(x, eps, rms)
    n = hat * pg + pb
    h = scale * residual + gate * n
    eh = (gate * pg).abs() * ehat + 4 * STEP * ((gate * n).abs() + (gate * hat * pg).abs() + (scale * residual).abs())
    return h, eh, hat, inv, ehat


def _double(x, residual, pg, pb, gate, gamma):
    x, residual, pg, gamma = (t.double() for t in (x, residual, pg, gamma))
    pb = torch.zeros_like(pg) if pb is None else pb.double()
    return x, residual, pg, pb, torch.ones_like(pg) if gate is None else gate.double(), gamma


def forward(x, residual, pg, pb, gate, scale, gamma, beta, eps, rms, u=0.0, least=0.0):
    """{"h", "y"} and their bounds; y is that of h before its rounding."""
    x, residual, pg, pb, gate, gamma = _double(x, residual, pg, pb, gate, gamma)
    beta = 0.0 if beta is None else beta.double()
    h, eh, *_ = _stream(x, residual, pg, pb, gate, scale, eps, rms)
    r = {"h": h, "bound_h": eh + 1.001 * u * h.abs() + least}
    hat, _, ehat = _norm(h, eps, rms, eh)
    r["y"] = hat * gamma + beta
    r["bound_y"] = (gamma.abs() * ehat + 4 * STEP * ((hat * gamma).abs() + r["y"].abs())
                    + 1.001 * u * r["y"].abs() + least)
    return r


def backward(x, residual, dh, dy, pg, pb, gate, scale, gamma, eps, rms, u=0.0, least=0.0):
    """{"dx", "dresidual", "dpost_gamma", "dpost_beta", "dgate", "dgamma",
    "dbeta"} and their bounds; dh or dy may be None."""
    x, residual, pg, pb, gate, gamma = _double(x, residual, pg, pb, gate, gamma)
    dh, dy = (torch.zeros_like(x) if t is None else t.double() for t in (dh, dy))
    rows = x.shape[0]
    h, eh, hat1, inv1, ehat1 = _stream(x, residual, pg, pb, gate, scale, eps, rms)
    hat2, inv2, ehat2 = _norm(h, eps, rms, eh)
    einv2 = inv2 * (hat2.abs() * eh).mean(1, keepdim=True)
    g2 = dy * gamma
    through, ethrough = _back(g2, STEP * g2.abs(), hat2, ehat2, inv2, rms, einv2)
    D = dh + through
    eD = ethrough + STEP * D.abs()
    g1 = D * gate * pg
    eg1 = (gate * pg).abs() * eD + 2 * STEP * g1.abs()
    dx, edx = _back(g1, eg1, hat1, ehat1, inv1, rms)
    r = {"dx": dx, "dresidual": scale * D}
    r["bound_dx"] = edx + 1.001 * u * dx.abs() + least
    r["bound_dresidual"] = abs(scale) * eD + (1.001 * u + STEP) * r["dresidual"].abs() + least
    deep = (rows / 256 + 40) * STEP

    def total(v, ev):
        return v.sum(0), ev.sum(0) + deep * v.abs().sum(0)

    s1, e1 = total(D * hat1, eD * hat1.abs() + D.abs() * ehat1)
    s2, e2 = total(D, eD)
    s3, e3 = total(dy * hat2, dy.abs() * ehat2)
    s4, e4 = total(dy, torch.zeros_like(dy))
    for name, v, e in (("dpost_gamma", gate * s1, gate.abs() * e1), ("dpost_beta", gate * s2, gate.abs() * e2),
                       ("dgate", pg * s1 + pb * s2, pg.abs() * e1 + pb.abs() * e2
                        + 2 * STEP * ((pg * s1).abs() + (pb * s2).abs())), ("dgamma", s3, e3), ("dbeta", s4, e4)):
        r[name], r["bound_" + name] = v, e + (1.001 * u + STEP) * v.abs() + least
    return r
