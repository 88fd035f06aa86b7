"""CPU: refusals of the token log probability and distillation entry points,
and their oracle against differences and closed forms."""

import math

import pytest
import torch

from eth_amd import _native as nat
from oracle.logit_rows import token_logprobs, topk_distill

P = 1 << 20
LOGP = dict(logits=P, ld=100, tokens=P, ignore=-100, logprob=P, entropy=P, stats=P, top=P, ids=P, k=5, ws=None, rows=4,
            vocab=100, bad=P, dtype=nat.ETH_BF16, stream=None)
LOGP_BWD = dict(logits=P, ld=100, tokens=P, ignore=-100, stats=P, entropy=P, dlogprob=P, dentropy=P, dz=P, ldd=100,
                rows=4, vocab=100, dtype=nat.ETH_BF16, stream=None)
DISTILL = dict(logits=P, ld=100, ids=P, teacher=P, teacher_dtype=nat.ETH_F32, k=8, tau=1.0, loss=P, stats=P, ws=None,
               rows=4, vocab=100, bad=P, dtype=nat.ETH_BF16, stream=None)
DISTILL_BWD = dict(logits=P, ld=100, ids=P, teacher=P, teacher_dtype=nat.ETH_F32, k=8, tau=1.0, stats=P, dloss=P, dz=P,
                   ldd=100, rows=4, vocab=100, bad=P, dtype=nat.ETH_BF16, stream=None)


@pytest.mark.parametrize("name,good,changes", [
    ("eth_token_logprobs_fwd", LOGP, [
        dict(dtype=3), dict(ld=99), dict(rows=0), dict(vocab=0), dict(vocab=2**24 + 1, ld=2**25), dict(k=-1), dict(k=129),
        dict(vocab=4, k=5), dict(logits=None), dict(tokens=None), dict(logprob=None), dict(stats=P + 4), dict(top=None),
        dict(ids=None), dict(bad=None), dict(logits=P + 1), dict(vocab=70000, ld=70000),
        dict(vocab=70000, ld=70000, ws=P + 8), dict(rows=2**31)]),
    ("eth_token_logprobs_bwd", LOGP_BWD, [
        dict(dtype=-1), dict(ld=99), dict(ldd=99), dict(rows=0), dict(dlogprob=None, dentropy=None), dict(entropy=None),
        dict(dz=None), dict(dz=P + 1), dict(stats=P + 4), dict(rows=2**31)]),
    ("eth_topk_distill_fwd", DISTILL, [
        dict(dtype=3), dict(teacher_dtype=3), dict(ld=99), dict(rows=0), dict(k=0), dict(k=257), dict(tau=0.0),
        dict(tau=-1.0), dict(tau=math.nan), dict(tau=math.inf), dict(ids=None), dict(teacher=None), dict(loss=None),
        dict(stats=None), dict(bad=None), dict(teacher=P + 2), dict(rows=2**31), dict(vocab=2**18, ld=2**18),
        dict(vocab=2**18, ld=2**18, ws=P + 4)]),
    ("eth_topk_distill_bwd", DISTILL_BWD, [
        dict(dtype=3), dict(ldd=99), dict(k=0), dict(tau=0.0), dict(dloss=None), dict(dz=None), dict(dz=P + 1),
        dict(stats=P + 4), dict(rows=2**31)]),
])
def test_c_entries_refuse_before_any_launch(name, good, changes):
    for change in changes:
        with pytest.raises(ValueError):
            nat.call(name, *(good | change).values())


def test_workspace_only_for_rows_of_several_parts():
    ws = lambda *a: nat.value("eth_token_logprobs_workspace", *a)  # noqa: E731
    assert ws(7, 65536, 20, nat.ETH_BF16) == 0 and ws(7, 32768, 20, nat.ETH_F32) == 0
    assert ws(7, 65537, 20, nat.ETH_F16) == 7 * 2 * (16 + 160)
    assert ws(7, 32769, 0, nat.ETH_F32) == 7 * 2 * 16
    assert ws(0, 65537, 20, nat.ETH_F16) == 0 and ws(7, 65537, 20, 5) == 0


def test_distillation_workspace_only_for_few_long_rows():
    ws = lambda *a: nat.value("eth_topk_distill_workspace", *a)  # noqa: E731
    assert ws(1, 98304, nat.ETH_BF16) == 0 and ws(129, 2**18, nat.ETH_BF16) == 0
    assert ws(1, 98305, nat.ETH_F16) == 4 * 8 and ws(1, 98304, nat.ETH_F32) == 6 * 8
    assert ws(64, 2**18, nat.ETH_BF16) == 64 * 8 * 8 and ws(128, 2**18, nat.ETH_BF16) == 128 * 4 * 8
    assert ws(1, 2**24, nat.ETH_F32) == 512 * 8 and ws(0, 2**18, nat.ETH_F32) == 0 and ws(1, 2**18, 7) == 0


def _slope(f, x, d):
    return (f(x + 1e-5 * d) - f(x - 1e-5 * d)) / 2e-5


def test_oracle_gradients_equal_differences():
    """Central differences in 64 bits with steps of 1e-5: off by about 1e-10."""
    gen = torch.Generator().manual_seed(4)
    z, d = (torch.randn(5, 23, generator=gen, dtype=torch.float64) * s for s in (2.0, 1.0))
    tokens = torch.tensor([3, -100, 22, 0, 7])
    g, h = (torch.randn(5, generator=gen, dtype=torch.float64) for _ in range(2))
    r = token_logprobs(z, tokens, 4, dlogprob=g, dentropy=h)

    def value(x):
        o = token_logprobs(x, tokens, 0)
        return (o["logprob"] * g + o["entropy"] * h).sum()

    assert abs(_slope(value, z, d) - (r["dz"] * d).sum()) < 1e-8
    assert (r["dz"][1] == 0).all() and (r["ids"][1] == -1).all()
    ids = torch.tensor([[1, 2, 5], [0, 0, 9], [-1, 3, 4], [-1, -1, -1], [22, 23, 0]])
    teacher = torch.randn(5, 3, generator=gen, dtype=torch.float64)
    for tau in (0.5, 1.0, 3.0):
        r = topk_distill(z, ids, teacher, tau, dloss=g)
        slope = _slope(lambda x: (topk_distill(x, ids, teacher, tau)["loss"] * g).sum(), z, d)
        assert abs(slope - (r["dz"] * d).sum()) < 1e-8
        assert r["loss"][3] == 0 and (r["dz"][3] == 0).all()


def test_oracle_closed_forms():
    z = torch.zeros(1, 8, dtype=torch.float64)
    r = token_logprobs(z, torch.tensor([5]), 3)
    assert abs(r["logprob"] + math.log(8)) < 1e-12 and abs(r["entropy"] - math.log(8)) < 1e-12
    assert r["ids"].tolist() == [[0, 1, 2]]
    # a teacher equal to the student over the whole vocabulary: no loss, no gradient
    z = torch.randn(1, 6, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    r = topk_distill(z, torch.arange(6)[None], z, 2.0, dloss=torch.ones(1))
    assert abs(r["loss"]) < 1e-12 and r["dz"].abs().max() < 1e-12
    # one entry: the cross entropy of its id
    r = topk_distill(z, torch.tensor([[4]]), torch.tensor([[0.3]], dtype=torch.float64), 1.0)
    assert abs(r["loss"] + torch.log_softmax(z, 1)[0, 4]) < 1e-12
