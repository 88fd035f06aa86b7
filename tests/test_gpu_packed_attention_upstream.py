"""GPU: the upstream gradient that autograd hands packed attention may be a part
of a larger one, at any offset: the gradients are those of the whole one's."""

import pytest
import torch

from eth_amd.model.functional import PackedCausalAttentionFn
from eth_amd.packed import PackedSequences
from tests.conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("before", [1, 4, 8])
def test_gradient_at_an_offset(cuda, before):
    announce(f"packed attention upstream gradient {before} elements in")
    lengths, n, m, hn = [40, 33], 4, 2, 64
    gen = torch.Generator().manual_seed(before)
    mixed = torch.randn(73, n + 2 * m, hn, generator=gen).bfloat16().to(cuda)
    dout = torch.randn(73, n * hn, generator=gen).bfloat16().to(cuda)
    packed = PackedSequences(lengths, device=cuda)
    grads = []
    for cut in (False, True):
        leaf = mixed.clone().requires_grad_(True)
        out = PackedCausalAttentionFn.apply(*torch.split(leaf, (n, m, m), dim=1), packed)
        g = dout
        if cut:
            other = torch.zeros(before, dtype=out.dtype, device=cuda, requires_grad=True)
            out = torch.cat([other, out.view(-1)])
            g = torch.cat([torch.ones_like(other), dout.view(-1)])
        grads.append(torch.autograd.grad(out, leaf, g)[0])
    torch.cuda.synchronize()
    assert torch.equal(*grads)
