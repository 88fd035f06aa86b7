"""GPU: gradients of the linear head's cross entropy for heads of more than 2 GiB,
whose vocabulary is taken in pieces within the reach of 32-bit offsets, against the
oracle in 64 bits with its bounds."""

import pytest
import torch

from eth_amd import kernels as K
from oracle.linear_xent import linear_xent
from tests.conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,H,V", [(70, 8192, 139001), (5, 16384, 66000)])
def test_heads_beyond_two_gibibytes(cuda, rows, H, V):
    announce(f"linear xent large head rows={rows} H={H} V={V}")
    gen = torch.Generator(device=cuda).manual_seed(V)
    randn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    h = randn(rows, H).bfloat16()
    w = torch.empty(V, H, dtype=torch.bfloat16, device=cuda)
    for at in range(0, V, 16384):
        w[at : at + 16384] = randn(min(16384, V - at), H) * (2.0 / H**0.5)
    whole = (2**31 - 1) // (2 * H) // 256 * 256
    assert V > whole
    labels = torch.randint(0, V, (rows,), generator=gen, device=cuda)
    labels[:4] = torch.tensor([whole - 1, whole, V - 1, 0], device=cuda)
    dloss = torch.rand(rows, generator=gen, device=cuda) + 0.5
    loss, lse = K.linear_xent_fwd(h, w, labels, torch.zeros(1, dtype=torch.int32, device=cuda))
    dh, dw = K.linear_xent_bwd(h, w, labels, lse, dloss)
    torch.cuda.synchronize()
    r = linear_xent(h, w, labels, -100, dloss, 2.0**-8, 2.0**-126)
    for name, got in (("loss", loss), ("dh", dh), ("dw", dw)):
        off = (got.double() - r[name]).abs()
        assert not got.isnan().any() and not (off > r["bound_" + name]).any(), f"{name}: {off.max():.3e} off"
