"""GPU: distillation over long rows against 64 bits, where rows are many (one
workgroup each) and where they are few (parts).

Tolerance.  A thread adds 8 vectors of 16 bytes a trip (64 terms of 16 bits, 32 of
fp32), its row's (or part's) trips of 512 threads' one after the other, then come
a tree of 9 levels, the waves (8), and the parts: n additions, each off by half a
step, n 2^-24 of the sum at the most.  An exponential of d < 0 is off by (|d| + 1)
2^-23 of itself, the logarithm and the two differences of a log probability by half
a step of its size each."""

import math

import pytest
import torch

from eth_amd import kernels as K
from tests.conftest import announce

pytestmark = pytest.mark.gpu


def _additions(rows, V, dtype):
    per = 4 if dtype == torch.float32 else 8
    trips = -(-V // (512 * 8 * per))
    parts = min(trips, 512 // rows) if trips >= 4 and 512 // rows >= 4 else 1
    return 8 * per + -(-trips // parts) + 1 + 9 + 8 + parts


def _log_bound(rows, V, dtype, spread, size):
    """Of a log probability of `size` under a row with sum p |z - max| = spread."""
    return _additions(rows, V, dtype) * 2.0**-24 + (1 + spread) * 2.0**-23 + 4 * (1 + size) * 2.0**-24


@pytest.mark.parametrize("rows,V,dtype", [
    (129, 2**22, torch.bfloat16), (129, 2**22, torch.float16), (130, 2**21, torch.float32), (128, 2**22, torch.bfloat16),
    (1, 2**24, torch.float32),
])
def test_sums_of_very_many_equal_terms(cuda, rows, V, dtype):
    """Logits of x, and among them a 0 in every thread's share of every trip, so
    that its maximum is 0: terms e^x, whose sum rounds the same way at many
    additions.  The loss of the one entry x is log(zeros + (V - zeros) e^x) - x."""
    announce(f"distill equal terms rows={rows} V={V} {dtype}")
    x = torch.tensor([-0.5, -0.703125, -1.0, -1.203125, -3.0, -1.5]).repeat(rows // 6 + 1)[:rows]
    z = x.to(dtype).to(cuda)[:, None].repeat(1, V)
    per = 16 // z.element_size()
    z.view(rows, -1, 8, 512, per)[:, :, 0, :, 0] = 0.0  # (trips of 8 vectors of 512 threads)
    zeros = V // (8 * per)
    ids, u = torch.ones(rows, 1, dtype=torch.int64, device=cuda), torch.zeros(rows, 1, device=cuda)
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    loss, _ = K.topk_distill_fwd(z, ids, u, 1.0, bad)
    x = x.double()  # (values of every type)
    want = torch.log(zeros + (V - zeros) * x.exp()) - x
    off = (loss.double().cpu() - want).abs()
    bound = _log_bound(rows, V, dtype, x.abs(), want)
    assert (off <= bound).all(), f"{off.max():.2e} off, {(off / bound).max():.2f} of the bound"


@pytest.mark.parametrize("rows,V,dtype,k,tau,pad", [
    (129, 131077, torch.bfloat16, 20, 1.0, 0), (140, 200003, torch.float16, 8, 2.0, 5), (130, 98305, torch.float32, 64, 0.5, 3),
])
def test_many_long_rows(cuda, rows, V, dtype, k, tau, pad):
    announce(f"distill many long rows {rows} x {V} {dtype} k={k} tau={tau}")
    gen = torch.Generator(device=cuda).manual_seed(V)
    buffer = (torch.randn(rows, V + pad, generator=gen, device=cuda) * 2.5).to(dtype)
    z = buffer[:, :V]
    u, ids = torch.topk(z.float() + torch.randn(rows, V, generator=gen, device=cuda), k, dim=1)
    ids, dloss = ids.contiguous(), torch.randn(rows, generator=gen, device=cuda)
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    loss, stats = K.topk_distill_fwd(z, ids, u, tau, bad)
    dz = K.topk_distill_bwd(z, ids, u, tau, stats, dloss, bad)
    d = z.double() / tau
    d = d - d.amax(1, keepdim=True)
    p = d.exp()
    total = p.sum(1, keepdim=True)
    p /= total
    logp = d - total.log()
    spread = -(p * d).sum(1)
    q = torch.softmax(u.double() / tau, 1)
    picked = logp.gather(1, ids)
    want = tau**2 * (q * (q.log() - picked)).sum(1)
    L = _log_bound(rows, V, dtype, spread, 0.0)
    # the entries' own weights: q of k terms with exponents as above, two logarithms
    size = (q * (1 + q.log().abs() + picked.abs())).sum(1)
    off = (loss.double() - want).abs()
    bound = tau**2 * (L + size * (k + 16) * 2.0**-23)
    assert (off <= bound).all(), f"{off.max():.2e} off, {(off / bound).max():.2f} of the bound"
    gt = (dloss.double() * tau)[:, None]
    target = torch.zeros_like(p).scatter_add_(1, ids, q)
    want = gt * (p - target)
    step = torch.finfo(dtype).eps / 2
    bound = gt.abs() * (p * (L[:, None] + (logp.abs() + 4) * 2.0**-22) + target * (k + 16) * 2.0**-22)
    bound += 1.001 * step * want.abs() + (2.0**-25 if dtype == torch.float16 else 2.0**-126)
    off = (dz.double() - want).abs()
    assert dz.shape == z.shape and not (off > bound).any(), f"{(off / bound).max():.2f} of the bound"
