"""GPU: gradients of the linear head's cross entropy where the label's probability
p is almost one, so that its dz, p - 1, is what the other columns' sum leaves.

h = c U and weights U or t U, U of 64 signs, c of 8 bits and t = 113/128: the logits
64 c and 64 c t are exact in fp32, with gaps of 7.5 c.  What is left to go wrong is the
row's statistics: its maximum is the label's logit up to fp32's rounding, whose
exponential is off by 2^-23; of the additions four meet the one that it stands for (of a
lane's columns and of a row's four lanes), 2^-24 each; so p - 1 is off by at most
2^-23 + 5 * 2^-24 < 2^-21 with what log, exp and their arguments add to a difference
of 2^-10 at most.  Another column's p is off by its share of that, by the rounding of lse
(log2: below 256, 2^-17) and by 2^-21."""

import pytest
import torch

from eth_amd import kernels as K
from tests.conftest import announce

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
STATISTICS, OTHERS = 2.0**-21, 2.0**-16
TYPES = [torch.bfloat16, torch.float16]


def _operands(cuda, rows, label, dtype, first=0, V=8):
    gen = torch.Generator().manual_seed(rows)
    u = torch.randint(0, 2, (64,), generator=gen) * 2.0 - 1.0
    c = 1.0 + ((torch.arange(rows) + first) % 116) / 128
    w = u * torch.where(torch.arange(V) == label, 1.0, 113 / 128)[:, None]
    h = c[:, None] * u
    assert (h.to(dtype) == h).all() and (w.to(dtype) == w).all()
    labels = torch.full((rows,), label)
    dloss = torch.rand(rows, generator=gen) + 0.5
    return h.to(dtype).to(cuda), w.to(dtype).to(cuda), labels.to(cuda), dloss.to(cuda)


def _check(h, w, labels, dloss, loss, dh, dw, u):
    """u: what a dz is off by, relative to it"""
    h, w, g = h.double(), w.double(), dloss.double()[:, None]
    z = h @ w.T
    other = torch.arange(w.shape[0], device=w.device) != labels[0]
    gap = (z - z[:, labels[:1]])[:, other].exp()
    rest = gap.sum(1, keepdim=True)
    assert rest.max() < 2.0**-7 and rest.min() > 2.0**-18
    assert ((loss.double() - rest.log1p()[:, 0]).abs() < STATISTICS).all()
    dz = torch.empty_like(z)
    dz[:, labels[0]] = (-rest / (1 + rest))[:, 0]
    dz[:, other] = gap / (1 + rest)
    off = (u + OTHERS) * dz.abs() + 2.0**-38
    off[:, labels[0]] += STATISTICS
    dz, off = dz * g, off * g
    # (sums of 8 columns and of the rows, in fp32: n roundings of 2^-23)
    for name, got, want, bound in (("dh", dh, dz @ w, off @ w.abs() + 8 * 2.0**-23 * dz.abs() @ w.abs()),
                                   ("dw", dw, dz.T @ h, off.T @ h.abs() + len(h) * 2.0**-23 * dz.abs().T @ h.abs())):
        if got.dtype != torch.float32:
            bound = bound + 1.001 * HALF_STEP[got.dtype] * want.abs() + 2.0**-25
        miss = (got.double() - want).abs()
        assert not got.isnan().any() and not (miss > bound).any(), (
            f"{name}: {miss.max():.3e} off, {(miss / bound).max():.2f} of the bound")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,label,first", [(1, 0, 115), (1, 5, 83), (1, 6, 40), (16, 3, 90), (48, 7, 7), (64, 2, 50),
                                              (116, 1, 0), (130, 6, 60), (300, 0, 0)])
def test_confident_rows(cuda, dtype, rows, label, first):
    announce(f"linear xent confident rows {dtype} rows={rows} first={first}")
    h, w, labels, dloss = _operands(cuda, rows, label, dtype, first)
    loss, lse = K.linear_xent_fwd(h, w, labels, torch.zeros(1, dtype=torch.int32, device=cuda))
    dw = torch.empty(w.shape, device=cuda)
    dh, _ = K.linear_xent_bwd(h, w, labels, lse, dloss, dweight=dw)
    # up to 64 rows dz is held in two parts
    _check(h, w, labels, dloss, loss, dh, dw, HALF_STEP[dtype] ** (2 if rows <= 64 else 1))


def test_statistics_of_the_forward(cuda):
    """lse is [2, rows]: the logits' logsumexp and the loss; other shapes are
    refused, and so is what else is wrong beside the right one."""
    announce("linear xent statistics")
    h, w, labels, dloss = _operands(cuda, 10, 4, torch.bfloat16)
    loss, lse = K.linear_xent_fwd(h, w, labels, torch.zeros(1, dtype=torch.int32, device=cuda))
    want = torch.logsumexp(h.double() @ w.double().T, 1)
    assert torch.equal(lse[1], loss) and ((lse[0].double() * 0.6931471805599453 - want).abs() < 2.0**-17).all()
    for bad in (lse[0], lse[:1], lse.t().contiguous(), lse.double(), lse[:, ::2].contiguous(), lse.cpu(), lse[:, :9],
                torch.cat([lse, lse])[::2]):
        with pytest.raises(ValueError):
            K.linear_xent_bwd(h, w, labels, bad, dloss)
    flat = torch.zeros(8 * 64 + 1, device=cuda)[1:].view(8, 64)
    for kw in (dict(dweight=torch.zeros(8, 64, device=cuda).bfloat16()), dict(dweight=torch.zeros(7, 64, device=cuda)),
               dict(accumulate=True), dict(dweight=flat), dict(dloss=dloss.half()), dict(dloss=dloss[:9])):
        with pytest.raises(ValueError):
            K.linear_xent_bwd(**(dict(hidden2d=h, weight=w, labels=labels, lse=lse, dloss=dloss) | kw))
