"""GPU: training passes whose saved tensors go to the host and back between
forward and backward give the gradients of those whose stay, bit for bit, also
where logits and projections are views of wider buffers."""

import pytest
import torch

from eth_amd.model.functional import PackedCausalAttentionFn, TokenLogprobsFn, TopkDistillFn
from eth_amd.packed import PackedSequences
from tests.conftest import announce

pytestmark = pytest.mark.gpu


def _with_and_without_offload(step):
    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logit_rows(cuda, dtype):
    announce(f"saved logit rows {dtype}")
    rows, V = 6, 1000
    gen = torch.Generator().manual_seed(1)
    buffer = torch.randn(rows, V + 47, generator=gen).to(dtype).to(cuda)
    tokens = torch.randint(0, V, (rows,), generator=gen).to(cuda)
    ids = torch.randint(0, V, (rows, 9), generator=gen).to(cuda)
    u = torch.randn(rows, 9, generator=gen).to(cuda)
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)

    def step():
        leaf = buffer.clone().requires_grad_(True)
        z = leaf[:, :V]
        logprob, entropy, _, _ = TokenLogprobsFn.apply(z, tokens, 3, bad)
        loss = TopkDistillFn.apply(z, ids, u, 2.0, bad)
        one = torch.autograd.grad((logprob + entropy).sum(), leaf, retain_graph=True)
        return *one, *torch.autograd.grad(loss.sum(), leaf)

    _with_and_without_offload(step)


@pytest.mark.parametrize("lengths,hn", [([70, 33], 64), ([1700, 33], 128)])
def test_packed_attention(cuda, lengths, hn):
    announce(f"saved packed attention {lengths} hn={hn}")
    n, m, rows = 4, 2, sum(lengths)
    gen = torch.Generator().manual_seed(2)
    mixed = torch.randn(rows, n + 2 * m, hn, generator=gen).bfloat16().to(cuda)
    dout = torch.randn(rows, n * hn, generator=gen).bfloat16().to(cuda)
    packed = PackedSequences(lengths, device=cuda)

    def step():
        leaf = mixed.clone().requires_grad_(True)
        out = PackedCausalAttentionFn.apply(*torch.split(leaf, (n, m, m), dim=1), packed)
        return out.detach(), *torch.autograd.grad(out, leaf, dout)

    _with_and_without_offload(step)
