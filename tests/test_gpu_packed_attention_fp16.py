"""GPU: fp16 gradients of packed attention over the range that gradients have
in training: small ones (a mean over many tokens, no loss scale) over long
sequences, where P is about 1/L and dS below fp16's normal numbers, and large
ones, where dS is above fp16's largest.

Tolerance, as a norm: the result's rounding (what rounding the 64-bit gradient
leaves), and beside it u = 2^-11 of the gradient's norm for the roundings of P
and dS to fp16 before the second product.  Each of those is off by at most u of
itself and is uniform in it, u / sqrt(3) in the mean square; the terms of a
gradient's sum are thousands with independent signs, so its error has u / sqrt(3)
of its norm, and the rounding of the stored output, which delta is formed of,
adds u / sqrt(3) of the small part that delta has of dP - delta.  That holds
for the whole gradient and for its last rows, whose P is smallest."""

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.packed import PackedSequences
from oracle.packed import packed_attention
from tests.conftest import announce

pytestmark = pytest.mark.gpu

U = 2.0**-11


def _grads(cuda, q, k, v, lengths, dout):
    packed = PackedSequences(lengths, device=cuda)
    q, k, v, dout = (t.to(cuda) for t in (q, k, v, dout))
    out, lse = K.packed_attention_fwd(q, k, v, packed)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    K.packed_attention_bwd(q, k, v, out, dout, lse, packed, *grads)
    return dict(zip(("dq", "dk", "dv"), grads))


def _check(got, ref, lengths):
    rows = sum(lengths)
    for name, g in got.items():
        g, want = g.double().cpu(), ref[name]
        assert g.isfinite().all(), name
        for part in (slice(0, rows), slice(lengths[0] // 2, lengths[0]), slice(lengths[0], rows)):
            w = want[part]
            bound = (w.half().double() - w).norm() + U * w.norm()
            off = (g[part] - w).norm()
            assert off <= bound, f"{name} rows {part.start}..{part.stop}: {off / w.norm():.2e}, {off / bound:.2f} of the bound"


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4])
@pytest.mark.parametrize("lengths,n,m,hn", [
    ([4000, 300], 2, 1, 64), ([4000, 300], 1, 1, 80), ([3000, 300], 4, 2, 128),  # split chains
    ([1000, 77], 2, 2, 64), ([1000, 77], 4, 1, 96), ([1000, 77], 2, 1, 128),  # whole ones
])
def test_small_gradients(cuda, lengths, n, m, hn, size):
    announce(f"fp16 gradients of size {size} {lengths} n={n} m={m} hn={hn}")
    gen = torch.Generator().manual_seed(hn)
    rows = sum(lengths)
    q, k, v = (torch.randn(rows, heads, hn, generator=gen).half() for heads in (n, m, m))
    dout = (torch.randn(rows, n * hn, generator=gen) * size).half()
    ref = packed_attention(*(t.double() for t in (q, k, v)), lengths, dout=dout.double().view(rows, n, hn))
    _check(_grads(cuda, q, k, v, lengths, dout), ref, lengths)


@pytest.mark.parametrize("lengths,n,m,hn", [
    ([1700, 300], 2, 1, 64), ([900, 77], 4, 2, 96), ([1700, 300], 2, 2, 128), ([900, 77], 4, 1, 128),
])
def test_large_gradients(cuda, lengths, n, m, hn):
    """dP of about 2^18: dS of the first rows is past fp16's largest number,
    dQ, dK and dV are not."""
    announce(f"fp16 gradients of large dout {lengths} n={n} m={m} hn={hn}")
    gen = torch.Generator().manual_seed(hn)
    rows = sum(lengths)
    q, k, v = (torch.randn(rows, heads, hn, generator=gen) for heads in (n, m, m))
    q, k, v = (q / 16).half(), (k / 16).half(), (v * 8).half()
    dout = (torch.randint(0, 2, (rows, n * hn), generator=gen) * 2 - 1).half() * 4096
    ref = packed_attention(*(t.double() for t in (q, k, v)), lengths, dout=dout.double().view(rows, n, hn))
    _check(_grads(cuda, q, k, v, lengths, dout), ref, lengths)


@pytest.mark.parametrize("hn", [64, 128])
def test_sizes_that_change_along_a_sequence(cuda, hn):
    """Gradients of sizes 1e-4, 64, 0 and 1 in blocks of a sequence; dQ of the
    first block, whose rows share no wave with others, is as exact as alone.  NaN
    in the sequence behind changes no bit."""
    announce(f"fp16 gradients of changing size hn={hn}")
    lengths, n, m = [900, 300], 2, 1
    gen = torch.Generator().manual_seed(hn + 1)
    rows = sum(lengths)
    q, k, v = (torch.randn(rows, heads, hn, generator=gen).half() for heads in (n, m, m))
    size = torch.tensor([1e-4, 64.0, 0.0, 1.0])[torch.arange(rows) // 130 % 4][:, None]
    dout = (torch.randn(rows, n * hn, generator=gen) * size).half()
    ref = packed_attention(*(t.double() for t in (q, k, v)), lengths, dout=dout.double().view(rows, n, hn))
    got = _grads(cuda, q, k, v, lengths, dout)
    _check(got, ref, lengths)
    first = ref["dq"][:128]
    off = (got["dq"][:128].double().cpu() - first).norm()
    assert off <= (first.half().double() - first).norm() + U * first.norm()
    dout[900:] = float("nan")
    again = _grads(cuda, q, k, v, lengths, dout)
    for name in got:
        assert torch.equal(again[name][:900], got[name][:900]), name
