"""CPU: refusals of the residual norm's entry points before any launch, its
structures, and its oracle against differences."""

import ctypes

import pytest
import torch

from eth_amd import _native as nat
from oracle import residual_norm as oracle

P = 1 << 20


def _desc(**change):
    d = nat.ResidualNormDesc()
    good = dict(post_gamma=P, post_beta=P, gate=P, gamma=P, beta=P, rows=4, cols=64, residual_scale=1.0, eps=1e-5, rms=0,
                dtype=nat.ETH_BF16)
    for k, v in (good | change).items():
        setattr(d, k, v)
    return d


BAD = [dict(dtype=nat.ETH_F32), dict(rows=-1), dict(rows=2**26), dict(rows=2**26 - 3), dict(cols=0), dict(cols=60), dict(cols=8200),
       dict(post_gamma=None), dict(gamma=None), dict(beta=None), dict(post_beta=None), dict(rms=1), dict(gate=P + 2),
       dict(gamma=P + 8), dict(eps=-1.0), dict(eps=float("inf")), dict(eps=float("nan")),
       dict(residual_scale=float("nan")), dict(residual_scale=float("inf"))]


def test_c_entries_refuse_before_any_launch():
    def fwd(desc, **change):
        args = dict(x=P, residual=P, h=P, y=P, stats=P, stream=None) | change
        nat.call("eth_residual_norm_fwd", ctypes.byref(desc) if desc else None, *args.values())

    def bwd(desc, table=None, **change):
        table = (nat.ResidualNormGrad * 5)() if table is None else table
        args = dict(x=P, residual=P, stats=P, dh=P, dy=P, dx=P, dres=P, grads=table, ws=P, stream=None) | change
        nat.call("eth_residual_norm_bwd", ctypes.byref(desc) if desc else None, *args.values())

    for call in (fwd, bwd):
        with pytest.raises(ValueError):
            call(None)
        for change in BAD:
            with pytest.raises(ValueError):
                call(_desc(**change))
    for change in (dict(x=None), dict(residual=None), dict(h=None), dict(y=None), dict(stats=None), dict(x=P + 2),
                   dict(y=P + 8)):
        with pytest.raises(ValueError):
            fwd(_desc(), **change)
    for change in (dict(x=None), dict(residual=None), dict(stats=None), dict(dh=None, dy=None), dict(grads=None), dict(ws=None),
                   dict(dh=P + 2), dict(dx=P + 8), dict(ws=P + 4)):
        with pytest.raises(ValueError):
            bwd(_desc(), **change)

    def table(*entries):
        t = (nat.ResidualNormGrad * 5)()
        for i, grad, fp32, accumulate in entries:
            t[i].grad, t[i].fp32, t[i].accumulate = grad, fp32, accumulate
        return t

    for desc, t in ((_desc(gate=None), table((2, P, 1, 0))), (_desc(rms=1, post_beta=None, beta=None), table((1, P, 1, 0))),
                    (_desc(rms=1, post_beta=None, beta=None), table((4, P, 0, 0))), (_desc(), table((0, P, 0, 1))),
                    (_desc(), table((0, P + 2, 1, 0))), (_desc(), table((0, P, 1, 0), (3, P, 1, 1)))):
        with pytest.raises(ValueError):
            bwd(desc, t)
    fwd(_desc(rows=0))  # (nothing to do)


def test_structures_and_workspace():
    assert ctypes.sizeof(nat.ResidualNormDesc) == 72 and ctypes.sizeof(nat.ResidualNormGrad) == 16
    ws = lambda *a: nat.value("eth_residual_norm_workspace", *a)  # noqa: E731
    assert ws(0, 64) == 0 and ws(1, 64) == 256 and ws(10**6, 2048) == 256 * 4 * 2048


@pytest.mark.parametrize("rms,gated", [(False, True), (True, False)])
def test_oracle_gradients_equal_differences(rms, gated):
    """Central differences in 64 bits with steps of 1e-5: off by about 1e-9."""
    gen = torch.Generator().manual_seed(2)
    randn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    v = dict(x=randn(3, 16), residual=randn(3, 16), pg=1 + 0.3 * randn(16), pb=None if rms else randn(16),
             gate=randn(16) if gated else None, gamma=1 + 0.3 * randn(16), beta=None if rms else randn(16))
    dh, dy = randn(3, 16), randn(3, 16)

    def value(v):
        r = oracle.forward(v["x"], v["residual"], v["pg"], v["pb"], v["gate"], 0.6, v["gamma"], v["beta"], 1e-5, rms)
        return (r["h"] * dh + r["y"] * dy).sum()

    r = oracle.backward(v["x"], v["residual"], dh, dy, v["pg"], v["pb"], v["gate"], 0.6, v["gamma"], 1e-5, rms)
    for key, name in (("x", "dx"), ("residual", "dresidual"), ("pg", "dpost_gamma"), ("pb", "dpost_beta"),
                      ("gate", "dgate"), ("gamma", "dgamma"), ("beta", "dbeta")):
        if v[key] is None:
            continue
        d = randn(*v[key].shape)
        slope = (value({**v, key: v[key] + 1e-5 * d}) - value({**v, key: v[key] - 1e-5 * d})) / 2e-5
        assert abs(slope - (r[name] * d).sum()) < 1e-7, name
