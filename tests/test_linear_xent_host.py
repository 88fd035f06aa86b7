"""CPU: refusals of the linear head's cross entropy entry points before any
launch, its workspace, and its oracle against differences."""

import pytest
import torch

from eth_amd import _native as nat
from oracle.linear_xent import linear_xent

P = 1 << 20
FWD = dict(h=P, ldh=64, w=P, ldw=64, labels=P, ignore=-100, loss=P, lse=P, ws=P, rows=4, hidden=64, vocab=100, bad=P,
           dtype=nat.ETH_BF16, stream=None)
BWD = dict(h=P, ldh=64, w=P, ldw=64, labels=P, ignore=-100, lse=P, dloss=P, dh=P, dw=P, dw_dtype=nat.ETH_BF16,
           accumulate=0, ws=P, rows=4, hidden=64, vocab=100, dtype=nat.ETH_BF16, stream=None)
BOTH = [dict(dtype=nat.ETH_F32), dict(dtype=5), dict(rows=0), dict(rows=2**21), dict(hidden=0), dict(hidden=60),
        dict(hidden=2**20, ldh=2**20, ldw=2**20), dict(vocab=0), dict(vocab=2**24 + 1), dict(ldh=56), dict(ldh=65),
        dict(ldw=56), dict(ldw=66), dict(h=None), dict(w=None), dict(labels=None), dict(ws=None), dict(ws=P + 16),
        dict(h=P + 8), dict(w=P + 2), dict(rows=2**20, ldh=1032), dict(rows=2**20, vocab=2**20)]


@pytest.mark.parametrize("name,good,changes", [
    ("eth_linear_xent_fwd", FWD, [*BOTH, dict(loss=None), dict(lse=None), dict(bad=None)]),
    ("eth_linear_xent_bwd", BWD, [*BOTH, dict(lse=None), dict(dloss=None), dict(dh=None, dw=None), dict(dh=P + 2),
                                  dict(dw=P + 8), dict(dw_dtype=nat.ETH_F16), dict(accumulate=1)]),
])
def test_c_entries_refuse_before_any_launch(name, good, changes):
    for change in changes:
        with pytest.raises(ValueError):
            nat.call(name, *(good | change).values())


def test_workspace():
    ws = lambda *a: nat.value("eth_linear_xent_workspace", *a)  # noqa: E731
    assert ws(0, 64, 100, 64, 0) == 0 and ws(4, 64, 100, 56, 3) == 0
    for rows, hidden, vocab in ((1, 64, 1), (2048, 2048, 50304), (8192, 4096, 50257), (2**21 - 1, 64, 262144)):
        for grads in (1, 2, 3):
            # a piece of dz, a copy of h, fp32 rows of dh for each split
            most = max(256 << 20, 512 * rows) + 2 * rows * hidden + 16 * 4 * rows * hidden + 28 * rows + 16 * 256
            assert 0 < ws(rows, hidden, vocab, hidden, grads) <= most
        assert ws(rows, hidden, vocab, hidden, 0) < 8 * (rows + 16) * (vocab / 32 + 8) + 12 * rows + 4096


def _slope(f, x, d):
    return (f(x + 1e-5 * d) - f(x - 1e-5 * d)) / 2e-5


def test_oracle_gradients_equal_differences():
    """Central differences in 64 bits with steps of 1e-5: off by about 1e-10."""
    gen = torch.Generator().manual_seed(4)
    h, w, dh, dw = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((5, 8), (13, 8), (5, 8), (13, 8)))
    labels = torch.tensor([3, -100, 12, 0, 40])
    g = torch.randn(5, generator=gen, dtype=torch.float64)
    r = linear_xent(h, w, labels, dloss=g)
    value = lambda a, b: (linear_xent(a, b, labels)["loss"] * g).sum()  # noqa: E731
    assert abs(_slope(lambda x: value(x, w), h, dh) - (r["dh"] * dh).sum()) < 1e-8
    assert abs(_slope(lambda x: value(h, x), w, dw) - (r["dw"] * dw).sum()) < 1e-8
    assert r["loss"][1] == 0 and (r["dh"][1] == 0).all()
    clamped = torch.nn.functional.cross_entropy(h @ w.T, labels.clamp_max(12), reduction="none")
    assert torch.allclose(r["loss"], clamped)
