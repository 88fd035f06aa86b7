"""GPU: fp16 gradients of adapters whose tiles differ in size.  A tile's products
x A^T and dy B carry a power of two of their own, so what one tile holds, zeros
alone included, takes no digits from the others' share of dA and dB."""

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.packed import AdapterRows
from oracle.adapters import adapter_linear
from tests.conftest import announce

pytestmark = pytest.mark.gpu

LENS, IDS = [32, 40, 70, 16, 9], [0, 0, 1, 1, 0]


def _operands(cuda, k, n, r, seed):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    o = dict(x=randn(167, k), w=randn(n, k) / k**0.5, a=randn(2, r, k) / k**0.5, b=randn(2, n, r) / r**0.5,
             dy=randn(167, n))
    # (nothing that a power of two used here takes out of fp16's normal numbers)
    o["b"] = torch.where(o["b"].abs() < 2.0**-2, 2.0**-2, o["b"])
    o["a"] = torch.where(o["a"].abs() < 2.0**-4, 2.0**-4, o["a"])
    return {name: t.half().to(cuda) for name, t in o.items()}


def _grads(o, rows):
    _, saved = K.adapter_linear_fwd(o["x"], o["w"], None, o["a"], o["b"], rows, save=True)
    da, db = (torch.empty(o[k].shape, device=o["x"].device) for k in ("a", "b"))
    K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, saved, False, (da, False), (db, False))
    return da, db


def _within(o, scales, got, what):
    """fp32 gradients against 64 bits: x A^T and dy B are off by half a step of fp16,
    2^-11 (the smallest by 2^-37 of the largest), the results by fp32's 2^-24."""
    counts = torch.tensor(LENS)
    of_row = torch.tensor(IDS).repeat_interleave(counts).to(o["x"].device)
    scale = torch.tensor(scales).repeat_interleave(counts).to(o["x"].device)
    r = adapter_linear(o["x"], o["w"], None, o["a"], o["b"], of_row, scale, o["dy"], 2.0**-11, 2.0**-126, 2.0**-37)
    for name, t in zip(("da", "db"), got):
        off, bound = (t.double() - r[name]).abs(), r["bound_" + name]
        assert not t.isnan().any() and not (off > bound).any(), (
            f"{what} {name}: {off.max():.3e} off, {(off / bound).nan_to_num(0.0).max():.2f} of the bound")


@pytest.mark.parametrize("k,n,r", [(128, 192, 16), (64, 320, 64), (200, 136, 128)])
def test_tiles_of_zeros(cuda, k, n, r):
    """Rows that are not scored have zero gradients, a segment may have scale
    zero, and padding zero inputs: beside them, smaller adapters give the same
    digits."""
    announce(f"adapter tiles of zeros k={k} n={n} r={r}")
    for zero, scales in (("dy", [1.0] * 5), ("x", [1.0] * 5), (None, [0.0, 1.0, 0.0, 2.0, 0.5])):
        rows = AdapterRows(LENS, IDS, scales, device=cuda)
        o = _operands(cuda, k, n, r, k + r)
        if zero:
            o[zero][:32], o[zero][72 : 72 + 64] = 0.0, 0.0
        want = _grads(o, rows)
        _within(o, scales, want, zero)
        small = dict(o, a=o["a"] * 2.0**-10, b=o["b"] * 2.0**-12)
        got = _grads(small, rows)
        _within(small, scales, got, f"small, {zero}")
        assert torch.equal(got[0], want[0] * 2.0**-12) and torch.equal(got[1], want[1] * 2.0**-10)
    # zeros alone
    o["dy"].zero_()
    assert all((g == 0).all() for g in _grads(o, rows))


@pytest.mark.parametrize("k,n,r", [(128, 192, 16), (64, 320, 64), (200, 136, 128)])
def test_small_tiles_beside_large_ones(cuda, k, n, r):
    """Where nothing else reaches an element, a small tile's share of it is what
    it is without the large tiles, bit for bit."""
    announce(f"adapter tiles of two sizes k={k} n={n} r={r}")
    scales = [2.0**20, 2.0**-20, 2.0**-20, 2.0**20, 2.0**-20]
    rows = AdapterRows(LENS, IDS, scales, device=cuda)
    large = torch.tensor([s > 1 for s in scales]).repeat_interleave(torch.tensor(LENS)).to(cuda)
    o = _operands(cuda, k, n, r, 3 * k + r)
    o["x"][large, : k // 2] = 0.0
    o["dy"][large, : n // 2] = 0.0
    da, db = _grads(o, rows)
    _within(o, scales, (da, db), "two sizes")
    alone_a = _grads(dict(o, dy=torch.where(large[:, None], 0.0, o["dy"])), rows)[0]
    alone_b = _grads(dict(o, x=torch.where(large[:, None], 0.0, o["x"])), rows)[1]
    assert torch.equal(da[:, :, : k // 2], alone_a[:, :, : k // 2]) and alone_a.abs().amin() > 0
    assert torch.equal(db[:, : n // 2], alone_b[:, : n // 2]) and alone_b.abs().amin() > 0
