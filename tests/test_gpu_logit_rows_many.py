"""GPU: logit rows whose workgroups have 2^32 threads and more in all, which one
launch cannot have: every row gives what it gives in a smaller call."""

import pytest
import torch

from eth_amd import kernels as K
from tests.conftest import announce

pytestmark = pytest.mark.gpu

ROWS, V = 2**24 + 1001, 3


def _parts():
    """(a block of rows that one launch takes, around the borders of the launches)"""
    for at in (0, 2**23 - 2500, 2**24 - 2500, ROWS - 5000):
        yield slice(at, at + 5000)


def test_token_logprobs(cuda):
    announce(f"token logprobs of {ROWS} rows")
    gen = torch.Generator(device=cuda).manual_seed(1)
    z = torch.randn(ROWS, V, generator=gen, device=cuda).bfloat16()
    tokens = torch.randint(0, V, (ROWS,), generator=gen, device=cuda)
    g, h = (torch.randn(ROWS, generator=gen, device=cuda) for _ in range(2))
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)

    def both(at):
        logprob, entropy, stats, top, ids = K.token_logprobs_fwd(z[at], tokens[at], 2, bad)
        dz = K.token_logprobs_bwd(z[at], tokens[at], stats, entropy, g[at], h[at], bad)
        return logprob, entropy, stats, top, ids, dz

    got = both(slice(0, ROWS))
    for at in _parts():
        for a, b in zip(got, both(at)):
            assert torch.equal(a[at], b)
    assert all(t.isfinite().all() for t in got)
    assert bad.item() == 0


def test_distillation(cuda):
    announce(f"distillation of {ROWS} rows")
    gen = torch.Generator(device=cuda).manual_seed(2)
    z = torch.randn(ROWS, V, generator=gen, device=cuda).half()
    ids = torch.randint(-1, V, (ROWS, 2), generator=gen, device=cuda)
    u, dloss = torch.randn(ROWS, 2, generator=gen, device=cuda), torch.randn(ROWS, generator=gen, device=cuda)
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)

    def both(at):
        loss, stats = K.topk_distill_fwd(z[at], ids[at], u[at], 2.0, bad)
        return loss, K.topk_distill_bwd(z[at], ids[at], u[at], 2.0, stats, dloss[at], bad)

    got = both(slice(0, ROWS))
    for at in _parts():
        for a, b in zip(got, both(at)):
            assert torch.equal(a[at], b)
    assert all(t.isfinite().all() for t in got)
    assert bad.item() == 0
