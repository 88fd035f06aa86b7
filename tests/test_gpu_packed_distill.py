"""The three operators as they are used together: a teacher scores packed
documents (packed attention, head, token log probabilities with their top
alternatives), a student learns from those alternatives (packed attention, head,
distillation) and its gradients come back through all of it.

Each stage is held to the oracle on the inputs that the GPU gave it, with the
bounds of its own tests (roundings of half a step; fp32 sums); autograd's
gradients equal the operators called by hand bit for bit."""

import math

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.model.functional import LinearFn, PackedCausalAttentionFn, TokenLogprobsFn, TopkDistillFn
from eth_amd.packed import PackedSequences
from oracle.logit_rows import token_logprobs, topk_distill
from oracle.packed import packed_attention
from tests.conftest import announce

pytestmark = pytest.mark.gpu

LENGTHS, ROWS, H, N, M, HN, V, TOP, TAU = [60, 1, 0, 70], 152, 64, 4, 2, 32, 504, 16, 2.0
USED = sum(LENGTHS)  # (the weight gradients take rows in whole groups of eight: 152)


def _weights(seed, cuda):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn((N + 2 * M) * HN, H, generator=gen) * 0.2
    head = torch.randn(V, N * HN, generator=gen) * 0.3
    return [w.bfloat16().to(cuda) for w in (qkv, head)]


def _logits(x, weights, packed):
    mixed = LinearFn.apply(x, weights[0], None).view(ROWS, N + 2 * M, HN)
    q, k, v = torch.split(mixed, (N, M, M), dim=1)
    out = PackedCausalAttentionFn.apply(q, k, v, packed)
    return LinearFn.apply(out, weights[1], None), out, mixed


def _inputs(cuda):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(ROWS, H, generator=gen).bfloat16().to(cuda)
    tokens = torch.randint(0, V, (ROWS,), generator=gen)
    tokens[USED:] = -100  # rows of no document are not scored
    return x, tokens.to(cuda), torch.zeros(1, dtype=torch.int32, device=cuda)


def _student(x, weights, packed, ids, top, bad):
    leaves = [t.detach().requires_grad_(True) for t in (x, *weights)]
    logits, out, mixed = _logits(leaves[0], leaves[1:], packed)
    loss = TopkDistillFn.apply(logits, ids, top, TAU, bad)
    grads = torch.autograd.grad(loss.sum() / USED, [*leaves, logits, out, mixed])
    return loss.detach(), logits.detach(), out.detach(), mixed.detach(), grads


def test_teacher_to_student(cuda):
    announce("teacher to student over packed documents")
    x, tokens, bad = _inputs(cuda)
    packed = PackedSequences(LENGTHS, total=ROWS, device=cuda)
    with torch.no_grad():
        tlogits, tout, tmixed = _logits(x, _weights(1, cuda), packed)
        logprob, entropy, top, ids = TokenLogprobsFn.apply(tlogits, tokens, TOP, bad)
    weights = _weights(2, cuda)
    loss, logits, out, mixed, grads = _student(x, weights, packed, ids, top, bad)
    dx, dqkv, dhead, dlogits, dout, dmixed = grads
    torch.cuda.synchronize()
    assert bad.item() == 0

    u = 2.0**-8
    split = lambda t: torch.split(t.double().cpu(), (N, M, M), dim=1)  # noqa: E731
    for got, m in ((tout, tmixed), (out, mixed)):
        r = packed_attention(*split(m), LENGTHS, u=u)
        off = (got.double().cpu().view(ROWS, N, HN) - r["out"]).abs()
        assert not (off > 1.25 * r["bound_out"] + 2.0**-22).any()
    r = token_logprobs(tlogits.double().cpu(), tokens.cpu(), TOP)
    assert torch.equal(ids.cpu(), r["ids"]) and (ids[USED:] == -1).all() and (top[USED:] == -math.inf).all()
    for got, want in ((logprob, r["logprob"]), (entropy, r["entropy"])):
        assert (got.double().cpu() - want).abs().max() < 2.0**-12 and (got[USED:] == 0).all()
    r = topk_distill(logits.double().cpu(), ids.cpu(), top.double().cpu(), TAU, torch.full((ROWS,), 1 / USED))
    assert (loss.double().cpu() - r["loss"]).abs().max() < 2.0**-12 and (loss[USED:] == 0).all()
    # (one rounding, and fp32 probabilities)
    off = (dlogits.double().cpu() - r["dz"]).abs()
    assert not (off > 1.01 * u * r["dz"].abs() + TAU / USED * 2.0**-14 * (r["logp"].exp() + r["q"])).any()

    # by hand
    g = torch.full((ROWS,), 1 / USED, device=cuda)
    _, stats = K.topk_distill_fwd(logits, ids, top, TAU, bad)
    by_hand = K.topk_distill_bwd(logits, ids, top, TAU, stats, g, bad)
    assert torch.equal(by_hand, dlogits)
    assert torch.equal(K.gemm(by_hand, weights[1]), dout)
    assert torch.equal(K.gemm(by_hand.t(), out, out_dtype=torch.bfloat16), dhead)
    q, k, v = torch.split(mixed, (N, M, M), dim=1)
    again, lse = K.packed_attention_fwd(q, k, v, packed)
    assert torch.equal(again, out)
    buffer = torch.full_like(mixed, math.nan)
    K.packed_attention_bwd(q, k, v, out, dout, lse, packed, *torch.split(buffer, (N, M, M), dim=1))
    assert torch.equal(buffer, dmixed)
    assert torch.equal(K.gemm(buffer.view(ROWS, -1), weights[0]), dx)
    assert torch.equal(K.gemm(buffer.view(ROWS, -1).t(), x, out_dtype=torch.bfloat16), dqkv)
    # rows of no document
    assert (dx[USED:] == 0).all() and (dlogits[USED:] == 0).all() and (out[USED:] == 0).all()

    # another first document leaves the others' losses and gradients as they were
    other = x.clone()
    other[:60] = other[:60].flip(0)
    loss2, _, _, _, grads2 = _student(other, weights, packed, ids, top, bad)
    assert torch.equal(loss2[60:], loss[60:]) and torch.equal(grads2[0][60:], dx[60:])
    assert not torch.equal(grads2[0][:60], dx[:60])


def test_self_distillation_is_a_fixed_point(cuda):
    """A student equal to its teacher, all alternatives given: p equals q up to
    fp32 sums, so the gradient is at most 2^-14 of what a probability weighs."""
    announce("self distillation")
    x, tokens, bad = _inputs(cuda)
    packed = PackedSequences(LENGTHS, total=ROWS, device=cuda)
    weights = _weights(1, cuda)
    weights[1] = weights[1][:128].contiguous()
    with torch.no_grad():
        logits = _logits(x, weights, packed)[0]
        _, _, top, ids = TokenLogprobsFn.apply(logits, tokens % 128, 128, bad)
    leaf = logits.detach().requires_grad_(True)
    loss = TopkDistillFn.apply(leaf, ids, top, 1.0, bad)
    (dz,) = torch.autograd.grad(loss.sum(), leaf)
    p = torch.softmax(logits.double(), 1)
    assert loss.abs().max() < 2.0**-12 and (dz.double().abs() <= 2.0**-14 * p + 2.0**-30).all()


def test_captured_training_step(cuda):
    """The student's whole step, backward pass included, captured once and
    replayed on new inputs."""
    announce("captured distillation step")
    x, tokens, bad = _inputs(cuda)
    packed = PackedSequences(LENGTHS, total=ROWS, device=cuda)
    weights = _weights(2, cuda)
    with torch.no_grad():
        _, _, top, ids = TokenLogprobsFn.apply(_logits(x, _weights(1, cuda), packed)[0], tokens, TOP, bad)
    inputs = [x, x.flip(0).contiguous(), x * 0.5]
    want = []
    for t in inputs:
        loss, _, _, _, grads = _student(t, weights, packed, ids, top, bad)
        want.append([loss, *grads[:3]])
    held = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _student(held, weights, packed, ids, top, bad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _, _, _, grads = _student(held, weights, packed, ids, top, bad)
        out = [loss, *grads[:3]]
    del loss, grads
    for i in (0, 1, 2, 1, 0):
        held.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(out, want[i]):
            assert torch.equal(got, w)
