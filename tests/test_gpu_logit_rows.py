"""GPU parity of token log probabilities (with entropy and top alternatives)
and of distillation from a teacher's top logits against the oracle in 64 bits
on the same logits.

Tolerances.  The kernels compute in fp32.  A row's sum of exponentials adds at
most 137 terms one after the other and a tree of 9 levels: relative error up to
146 * 2^-24 < 2^-16; an exponential of d < 0 is off by |d| 2^-23 + 2^-23
relatively.  With d weighted by probabilities (the oracle's "spread" a = sum p
|z - max|), log s is off by at most 2^-16 + (1 + a) 2^-22 =: L, a log probability
by L + |logp| 2^-22, the entropy by L + a (2^-15 + ...) < L + (1 + a) 2^-14.
Gradients add one rounding of half a step of the logits' type."""

import math
import threading

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.model.functional import TokenLogprobsFn, TopkDistillFn
from oracle.logit_rows import token_logprobs, topk_distill
from tests.conftest import announce

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
LEAST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25, torch.float32: 2.0**-126}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _bad(cuda):
    return torch.zeros(1, dtype=torch.int32, device=cuda)


def _logits(rows, V, dtype, seed, pad=0):
    gen = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, V + pad, generator=gen) * 2.5
    hot = torch.randint(0, V, (rows, 6), generator=gen)
    z.scatter_add_(1, hot, torch.randn(rows, 6, generator=gen).abs() * 5)
    return z.to(dtype), gen


def _same_or_within(got, want, bound, what):
    got = got.double().cpu()
    special = ~want.isfinite()
    assert torch.equal(got[special].nan_to_num(nan=7.0), want[special].nan_to_num(nan=7.0)), what
    off = (got - want).abs()[~special]
    bound = bound.expand_as(want)[~special]
    assert not (off > bound).any() and not got[~special].isnan().any(), (
        f"{what}: {off.max():.3e} off, {(off / bound).max():.2f} of the bound")


def _check_logp(z, tokens, top_k, got, g=None, h=None, dz=None, ignore=-100):
    """z: the CPU logits that the GPU had."""
    r = token_logprobs(z.double(), tokens, top_k, ignore, g, h)
    L = 2.0**-16 + (1 + r["spread"]) * 2.0**-22
    logprob, entropy, top, ids = got
    assert torch.equal(ids.cpu(), r["ids"])
    small = lambda x: torch.where(x.isfinite(), x.abs(), 0.0) * 2.0**-22  # noqa: E731
    _same_or_within(logprob, r["logprob"], L + small(r["logprob"]), "logprob")
    _same_or_within(top, r["top"], L[:, None] + small(r["top"]), "top")
    E = L + (1 + r["spread"]) * 2.0**-14
    want = torch.where(r["logprob"].isnan(), math.nan, r["entropy"])
    _same_or_within(entropy, want, E, "entropy")
    if dz is not None:
        g, h = (torch.zeros(z.shape[0]) if x is None else x for x in (g, h))
        lp = torch.where(r["logp"].isfinite(), r["logp"], 0.0)
        p = torch.where(r["logp"].isfinite(), r["logp"].exp(), 0.0)
        g, h = g.double().abs()[:, None], h.double().abs()[:, None]
        H = r["entropy"][:, None].abs()
        bound = (p * (L[:, None] + (1 + lp.abs()) * 2.0**-21) * (g + h * (lp.abs() + H))
                 + p * h * (E + L)[:, None] + (p * h * lp.abs() + g) * 2.0**-21)
        _same_or_within(dz, r["dz"], bound + HALF_STEP[z.dtype] * r["dz"].abs() * 1.001 + LEAST[z.dtype], "dz")


def _run_logp(z, tokens, top_k, bad, g, h, ignore=-100):
    logprob, entropy, stats, top, ids = K.token_logprobs_fwd(z, tokens, top_k, bad, ignore)
    dz = K.token_logprobs_bwd(z, tokens, stats, entropy, g, h, bad, ignore)
    return (logprob, entropy, top, ids), dz


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,top_k,pad", [
    (1, 1, 1, 0), (2, 2, 2, 3), (3, 7, 4, 0), (5, 8, 8, 0), (2, 9, 0, 1), (4, 127, 127, 0), (3, 1000, 128, 5),
    (2, 4097, 20, 0), (3, 16385, 5, 0), (2, 32001, 64, 7), (1, 50304, 5, 0), (2, 50257, 20, 47), (1, 65537, 128, 0),
    (2, 70001, 33, 2),
])
def test_token_logprobs(cuda, dtype, rows, V, top_k, pad):
    announce(f"token logprobs {dtype} rows={rows} V={V} k={top_k} pad={pad}")
    z, gen = _logits(rows, V, dtype, rows * V + top_k, pad)
    tokens = torch.randint(0, V, (rows,), generator=gen)
    g, h = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)
    zd = z.to(cuda)[:, :V]
    bad = _bad(cuda)
    got, dz = _run_logp(zd, tokens.to(cuda), top_k, bad, g.to(cuda), h.to(cuda))
    torch.cuda.synchronize()
    _check_logp(z[:, :V], tokens, top_k, got, g, h, dz)
    assert bad.item() == 0


def _special_rows(V, dtype):
    """Rows where a mask leaves nothing or little, equal logits, and orders of
    the values."""
    low = torch.finfo(dtype).min
    gen = torch.Generator().manual_seed(V)
    base = (torch.randn(V, generator=gen) * 2).to(dtype)
    rows = {
        "all -inf": torch.full((V,), -math.inf, dtype=dtype),
        "all lowest": torch.full((V,), low, dtype=dtype),
        "all equal": torch.full((V,), 1.5, dtype=dtype),
        "zeros of both signs": torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0).to(dtype),
        "one finite": torch.full((V,), -math.inf, dtype=dtype).index_fill_(0, torch.tensor([V // 2]), 2.0),
        "few finite": torch.where(torch.arange(V) % max(V // 7, 1) == 1, base, torch.tensor(-math.inf, dtype=dtype)),
        "few above the lowest": torch.where(torch.arange(V) % max(V // 7, 1) == 1, base, torch.tensor(low, dtype=dtype)),
        "ascending": base.sort()[0],
        "descending": base.sort(descending=True)[0],
        "two values": torch.where(torch.arange(V) % 3 == 0, 1.0, 0.5).to(dtype),
        "-inf at the end": torch.cat([base[: V // 2], torch.full((V - V // 2,), -math.inf, dtype=dtype)]),
        "large offset": (base + 1000).to(dtype),
    }
    return list(rows), torch.stack(list(rows.values()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,top_k", [(40, 20), (5000, 128), (40001, 17), (66000, 3)])
def test_token_logprobs_special_rows(cuda, dtype, V, top_k):
    names, z = _special_rows(V, dtype)
    announce(f"token logprobs special rows {dtype} V={V} k={top_k}: {names}")
    gen = torch.Generator().manual_seed(1)
    tokens = torch.full((len(names),), V // 2)
    g, h = torch.randn(len(names), generator=gen), torch.randn(len(names), generator=gen)
    got, dz = _run_logp(z.to(cuda), tokens.to(cuda), top_k, _bad(cuda), g.to(cuda), h.to(cuda))
    _check_logp(z, tokens, top_k, got, g, h, dz)
    assert (dz[0] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 70001])
def test_token_logprobs_non_finite(cuda, dtype, V):
    """NaN and +inf make their own row NaN and no other; NaN sorts first."""
    announce(f"token logprobs non-finite {dtype} V={V}")
    z, _ = _logits(4, V, dtype, 2)
    z[0, V - 1] = math.nan
    z[1, 17] = math.inf
    z[2, [5, 290]] = torch.tensor([math.nan, -math.nan], dtype=dtype)
    tokens = torch.tensor([3, 17, 5, 9])
    got, dz = _run_logp(z.to(cuda), tokens.to(cuda), 6, _bad(cuda), torch.ones(4, device=cuda), None)
    _check_logp(z, tokens, 6, got)
    assert dz[:3].isnan().any(1).all() and dz[3].isfinite().all()


def test_token_logprobs_ignored_and_out_of_range(cuda):
    """Ignored rows and rows without upstream gradient are not read (NaN in
    them reaches nothing); other bad ids are clamped and flagged."""
    announce("token logprobs ignored rows")
    for V in (1000, 70000):
        z, _ = _logits(5, V, torch.bfloat16, 3)
        z[1], z[3] = math.nan, math.nan
        tokens = torch.tensor([4, -100, V - 1, -100, 0])
        bad = _bad(cuda)
        g, h = torch.tensor([1.0, math.nan, 0.0, 1.0, -2.0]), torch.tensor([0.5, 1.0, 0.0, 1.0, 0.0])
        got, dz = _run_logp(z.to(cuda), tokens.to(cuda), 3, bad, g.to(cuda), h.to(cuda))
        clean = torch.where(torch.tensor([1, 0, 1, 0, 1])[:, None] > 0, z, torch.zeros_like(z))
        _check_logp(clean, tokens, 3, got, torch.nan_to_num(g), h, dz)
        assert (dz[1:4] == 0).all() and bad.item() == 0
        other, _ = _run_logp(z.to(cuda), torch.tensor([4, 7, V - 1, 7, 0]).to(cuda), 3, bad, g.to(cuda), h.to(cuda), 7)
        assert all(torch.equal(a, b) for a, b in zip(got, other))
        wild = torch.tensor([-1, -100, V, -100, 2**40])
        got, _ = _run_logp(z.to(cuda), wild.to(cuda), 3, bad, g.to(cuda), h.to(cuda))
        assert bad.item() == 1
        _check_logp(clean, torch.tensor([0, -100, V - 1, -100, V - 1]), 3, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,k,tau,teacher,pad", [
    (1, 1, 1, 1.0, torch.float32, 0), (3, 7, 7, 0.5, torch.float32, 1), (2, 130, 20, 2.0, torch.bfloat16, 0),
    (3, 4099, 64, 1.0, torch.float16, 5), (2, 50257, 256, 4.0, torch.float32, 47), (1, 50304, 8, 1.0, torch.float32, 0),
    (2, 70001, 100, 0.7, torch.float32, 0), (3, 98305, 20, 1.0, torch.float32, 3), (1, 2**20 + 5, 256, 2.0, torch.bfloat16, 0),
])
def test_topk_distill(cuda, dtype, rows, V, k, tau, teacher, pad):
    announce(f"distill {dtype} rows={rows} V={V} k={k} tau={tau} {teacher}")
    z, gen = _logits(rows, V, dtype, V + k, pad)
    full = z[:, :V].float() + torch.randn(rows, V, generator=gen)
    u, ids = (x.contiguous() for x in torch.topk(full, min(k, V), dim=1))
    u = u.to(teacher)
    dloss = torch.randn(rows, generator=gen)
    _distill_case(cuda, z.to(cuda)[:, :V], z[:, :V], ids, u, tau, dloss)


def _distill_case(cuda, zd, z, ids, u, tau, dloss, bad_expected=0):
    bad = _bad(cuda)
    loss, stats = K.topk_distill_fwd(zd, ids.to(cuda), u.to(cuda), tau, bad)
    dz = K.topk_distill_bwd(zd, ids.to(cuda), u.to(cuda), tau, stats, dloss.to(cuda), bad)
    torch.cuda.synchronize()
    r = topk_distill(z.double(), ids, u.double(), tau, dloss)
    _same_or_within(loss, r["loss"], tau**2 * (r["size"] * 2.0**-15 + 2.0**-20), "loss")
    lp = torch.where(r["logp"].isfinite(), r["logp"], 0.0)
    p = torch.where(r["logp"].isfinite(), r["logp"].exp(), 0.0)
    gt = dloss.double().abs()[:, None] * tau
    bound = gt * (p * (2.0**-15 + lp.abs() * 2.0**-21) + r["q"] * 2.0**-18)
    _same_or_within(dz, r["dz"], bound + HALF_STEP[z.dtype] * r["dz"].abs() * 1.001 + LEAST[z.dtype], "dz")
    assert bad.item() == bad_expected
    return loss, dz


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 9001, 100003])
def test_topk_distill_special_rows(cuda, dtype, V):
    """Rows without entries, with absent, repeated and masked ones, masked
    students, equal logits, a mask of the lowest value."""
    announce(f"distill special rows {dtype} V={V}")
    low = torch.finfo(dtype).min
    z, _ = _logits(10, V, dtype, 6)
    ids = torch.tensor([[3, 7, 9, 11]]).repeat(10, 1)
    u = torch.tensor([[2.0, 1.0, 0.5, -1.0]]).repeat(10, 1)
    ids[0] = -1
    ids[1] = torch.tensor([-1, V - 1, -5, 0])
    ids[2] = torch.tensor([3, 3, 9, 3])  # the same id three times
    u[3] = -math.inf
    u[4, 1:] = -math.inf
    z[5] = low
    z[6, 20:] = -math.inf
    z[7] = 0.25
    z[8, 20:] = low
    u[9] = torch.finfo(torch.float32).min  # equal entries all the same
    z[0], z[3] = math.nan, math.inf  # rows that are not read
    dloss = torch.tensor([1.0, -2.0, 0.5, 3.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.7])
    loss, dz = _distill_case(cuda, z.to(cuda), z, ids, u, 1.0, dloss)
    assert loss[0] == 0 and loss[3] == 0 and (dz[[0, 3]] == 0).all()
    # a zero upstream gradient, a student of -inf alone, one without the teacher's tokens
    z[0], z[3] = -math.inf, 1.0
    z[6, 3] = -math.inf
    ids[0], u[3] = torch.tensor([3, 7, 9, 11]), 0.0
    dloss[7] = 0.0
    loss, dz = _distill_case(cuda, z.to(cuda), z, ids, u, 2.0, dloss)
    assert loss[0] == math.inf and loss[6] == math.inf and (dz[[0, 7]] == 0).all()
    # ids past the vocabulary are flagged and left out
    ids[8] = torch.tensor([V, 7, 2**40, 11])
    _distill_case(cuda, z.to(cuda), z, ids, u, 1.0, dloss, bad_expected=1)
    # NaN stays in its row
    z[1, 5], u[2, 0] = math.nan, math.nan
    bad = _bad(cuda)
    ids[8] = -1
    loss, stats = K.topk_distill_fwd(z.to(cuda), ids.to(cuda), u.to(cuda), 1.0, bad)
    dz = K.topk_distill_bwd(z.to(cuda), ids.to(cuda), u.to(cuda), 1.0, stats, dloss.to(cuda), bad)
    assert loss.isnan().nonzero().flatten().tolist() == [1, 2] and dz[[4, 5, 9]].isfinite().all()


def test_offsets_past_32_bits(cuda):
    """90000 rows of 50304 logits (9 GiB): rows past 2^31 and 2^32 elements
    give what they give alone."""
    announce("logit rows past 32 bits")
    rows, V = 90000, 50304
    z = torch.zeros(rows, V, dtype=torch.bfloat16, device=cuda)
    some = torch.tensor([0, 42690, 85381, rows - 1], device=cuda)
    part = (torch.randn(4, V, generator=torch.Generator().manual_seed(1)) * 2).bfloat16().to(cuda)
    z[some] = part
    tokens = torch.full((rows,), -100, device=cuda)
    tokens[some] = 77
    g = torch.ones(rows, device=cuda)
    bad = _bad(cuda)
    got, dz = _run_logp(z, tokens, 4, bad, g, g)
    alone, dalone = _run_logp(part, tokens[some], 4, bad, g[:4], g[:4])
    assert all(torch.equal(a[some], b) for a, b in zip(got, alone)) and torch.equal(dz[some], dalone)
    del dz
    ids, u = torch.full((rows, 2), -1, device=cuda), torch.zeros(rows, 2, device=cuda)
    ids[some] = torch.tensor([5, 50303], device=cuda)
    loss, stats = K.topk_distill_fwd(z, ids, u, 1.0, bad)
    dz = K.topk_distill_bwd(z, ids, u, 1.0, stats, g, bad)
    loss4, stats4 = K.topk_distill_fwd(part, ids[some], u[:4], 1.0, bad)
    dz4 = K.topk_distill_bwd(part, ids[some], u[:4], 1.0, stats4, g[:4], bad)
    assert torch.equal(loss[some], loss4) and torch.equal(dz[some], dz4) and bad.item() == 0


def test_autograd_streams_and_replays(cuda):
    """Through autograd with any leading shape, with one upstream gradient or
    none, on two streams at once, and captured and replayed on new inputs."""
    announce("logit rows autograd, streams, graphs")
    V, bad = 70001, _bad(cuda)
    sets = []
    for seed in range(3):
        z, gen = _logits(6, V, torch.bfloat16, seed)
        u, ids = torch.topk(z.float() + torch.randn(6, V, generator=gen), 20, dim=1)
        tokens = torch.randint(0, V, (2, 3), generator=gen)
        sets.append([x.to(cuda) for x in (z.view(2, 3, V), tokens, ids.view(2, 3, 20), u.view(2, 3, 20))])

    def step(z, tokens, ids, u):
        leaf = z.detach().requires_grad_(True)
        logprob, entropy, top, top_ids = TokenLogprobsFn.apply(leaf, tokens, 7, bad)
        loss = TopkDistillFn.apply(leaf, ids, u, 2.0, bad)
        assert not top.requires_grad and top.shape == (2, 3, 7) and top_ids.dtype == torch.int64
        (dz,) = torch.autograd.grad((logprob + 0.3 * entropy + loss).sum(), leaf)
        return [logprob.detach(), entropy.detach(), top, top_ids, loss.detach(), dz]

    want = [step(*s) for s in sets]
    z, tokens, ids, u = sets[0]
    one = torch.ones(6, device=cuda)
    _, _, stats, _, _ = K.token_logprobs_fwd(z.view(6, V), tokens.view(6), 0, bad)
    entropy = want[0][1].view(6)
    d1 = K.token_logprobs_bwd(z.view(6, V), tokens.view(6), stats, entropy, one, 0.3 * one, bad)
    _, stats2 = K.topk_distill_fwd(z.view(6, V), ids.view(6, 20), u.view(6, 20), 2.0, bad)
    d2 = K.topk_distill_bwd(z.view(6, V), ids.view(6, 20), u.view(6, 20), 2.0, stats2, one, bad)
    assert torch.equal(want[0][5].view(6, V), d1 + d2)
    leaf = z.detach().requires_grad_(True)
    for pick, (g, h) in ((0, (one, None)), (1, (None, one))):
        out = TokenLogprobsFn.apply(leaf, tokens, 0, bad)[pick]
        bad.zero_()  # (a flag that is read and cleared between the passes)
        (dz,) = torch.autograd.grad(out.sum(), leaf)
        assert torch.equal(dz.view(6, V), K.token_logprobs_bwd(z.view(6, V), tokens.view(6), stats, entropy, g, h, bad))
    # a broadcast row: one gradient, the sum of its copies'
    wide = torch.randn(1, 64, device=cuda).requires_grad_(True)
    lp = TokenLogprobsFn.apply(wide.expand(3, 64), torch.tensor([1, 2, 3], device=cuda), 0, bad)[0]
    (dz,) = torch.autograd.grad(lp.sum(), wide)
    p = torch.softmax(wide.detach().double(), 1)
    p = -3 * p
    p[0, 1:4] += 1
    assert dz.shape == (1, 64) and (dz.double() - p).abs().max() < 2.0**-16
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(step(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    held = [x.clone() for x in sets[0]]

    def captured():
        z, tokens, ids, u = held
        z, tokens, ids, u = z.view(6, V), tokens.view(6), ids.view(6, 20), u.view(6, 20)
        logprob, entropy, stats, top, top_ids = K.token_logprobs_fwd(z, tokens, 7, bad)
        loss, stats2 = K.topk_distill_fwd(z, ids, u, 2.0, bad)
        d1 = K.token_logprobs_bwd(z, tokens, stats, entropy, one, 0.3 * one, bad)
        return logprob, entropy, top, top_ids, loss, d1 + K.topk_distill_bwd(z, ids, u, 2.0, stats2, one, bad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured()
    for s in (0, 1, 2, 0):
        for a, b in zip(held, sets[s]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want[s]):
            assert torch.equal(a.flatten(), b.flatten())
        step(*sets[(s + 1) % 3])
    empty = TokenLogprobsFn.apply(torch.zeros(0, V, device=cuda), torch.zeros(0, dtype=torch.int64, device=cuda), 2, bad)
    assert [tuple(x.shape) for x in empty] == [(0,), (0,), (0, 2), (0, 2)]


def test_refusals(cuda):
    announce("logit rows refusals")
    bad = _bad(cuda)
    z = torch.zeros(4, 100, dtype=torch.bfloat16, device=cuda)
    t = torch.zeros(4, dtype=torch.int64, device=cuda)
    K.token_logprobs_fwd(z, t, 5, bad)
    for args in [(z, t, 101, bad), (z, t, -1, bad), (z, t[:3], 5, bad), (z, t.int(), 5, bad), (z.double(), t, 5, bad),
                 (z.t(), t, 5, bad), (z[:1].expand(4, 100), t, 5, bad), (z.cpu(), t, 5, bad), (z, t.cpu(), 5, bad),
                 (z, t, 5, bad.float()), (z, t, 5, bad.cpu()), (z[0], t, 5, bad)]:
        with pytest.raises(ValueError):
            K.token_logprobs_fwd(*args)
    with pytest.raises(ValueError):
        K.token_logprobs_fwd(torch.zeros(4, 200, dtype=torch.bfloat16, device=cuda), t, 129, bad)
    logprob, entropy, stats, _, _ = K.token_logprobs_fwd(z, t, 0, bad)
    for args in [(stats, entropy, None, None), (stats[:, :1], entropy, logprob, None), (stats, entropy[:3], logprob, None),
                 (stats, entropy, logprob.double(), None), (stats, entropy, logprob, logprob[:3])]:
        with pytest.raises(ValueError):
            K.token_logprobs_bwd(z, t, *args, bad)
    ids, u = torch.zeros(4, 3, dtype=torch.int64, device=cuda), torch.zeros(4, 3, device=cuda)
    loss, stats = K.topk_distill_fwd(z, ids, u, 1.0, bad)
    for args in [(z, ids[:3], u[:3], 1.0), (z, ids, u[:, :2], 1.0), (z, ids.int(), u, 1.0), (z, ids, u.double(), 1.0),
                 (z, ids, u, 0.0), (z, ids, u, -1.0), (z, ids, u, math.inf), (z, ids, u, math.nan),
                 (z, ids[:, :0], u[:, :0], 1.0), (z, ids.t().contiguous().t(), u, 1.0),
                 (z, ids, u.t().contiguous().t(), 1.0), (z, ids.cpu(), u, 1.0),
                 (z, ids.repeat(1, 86), u.repeat(1, 86), 1.0)]:
        with pytest.raises(ValueError):
            K.topk_distill_fwd(*args, bad)
        with pytest.raises(ValueError):
            K.topk_distill_bwd(*args, stats, loss, bad)
    for s, d in ((stats[:3], loss), (stats, loss[:3]), (stats, loss.half())):
        with pytest.raises(ValueError):
            K.topk_distill_bwd(z, ids, u, 1.0, s, d, bad)
    with pytest.raises(ValueError):
        TokenLogprobsFn.apply(z, t[:2], 0, bad)
    with pytest.raises(ValueError):
        TopkDistillFn.apply(z, ids[:2], u[:2], 1.0, bad)


def test_whole_numbers_and_a_temperature_tensor(cuda):
    announce("logit rows arguments")
    bad = _bad(cuda)
    z = torch.randn(4, 100, device=cuda)
    t = torch.zeros(4, dtype=torch.int64, device=cuda)
    for changes in (dict(top_k=2.5), dict(ignore_index=0.5)):
        with pytest.raises(TypeError):
            K.token_logprobs_fwd(z, t, **(dict(top_k=2, bad_flag=bad) | changes))
    ids, u = torch.arange(12, device=cuda).view(4, 3), torch.randn(4, 3, device=cuda)
    grads = []
    for temperature in (2.0, torch.tensor(2.0), torch.tensor(2.0, device=cuda)):
        leaf = z.clone().requires_grad_(True)
        loss = TopkDistillFn.apply(leaf, ids, u, temperature, bad)
        if isinstance(temperature, torch.Tensor):
            temperature.fill_(5.0)
        grads.append(torch.autograd.grad(loss.sum(), leaf)[0])
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("top_k", [128, 127, 20, 1])
@pytest.mark.parametrize("V", [262144, 2**21 + 3, 2**24])
def test_alternatives_joined_from_many_parts(cuda, V, top_k):
    """The largest logits spread over the parts of a long row in shares of every
    size (1, 2, 4, .. of a part, all in one, one in each), among equal ones and
    among random ones: the ids of a stable sort, and its log probabilities."""
    announce(f"token logprobs joined V={V} k={top_k}")
    gen = torch.Generator().manual_seed(V % 1000 + top_k)
    z = torch.zeros(5, V)
    z[1] = torch.randn(V, generator=gen)
    z[2, V // 2 : V // 2 + 300] = 4.0 + torch.randn(300, generator=gen).abs()
    z[3, :: max(1, V // 200)] += 3.0
    at, share = 0, 64
    while share:
        for _ in range(max(1, 64 // share)):  # 64 in all of every share
            z[4, at : at + share] = 5.0 + torch.randn(share, generator=gen).abs()
            at += 32768
            if at + 64 > V:
                break
        if at + 64 > V:
            break
        share //= 2
    tokens, bad = torch.zeros(5, dtype=torch.int64), _bad(cuda)
    got = K.token_logprobs_fwd(z.to(cuda), tokens.to(cuda), top_k, bad)
    for row in range(5):
        order = torch.sort(z[row], descending=True, stable=True).indices[:top_k]
        assert torch.equal(got[4][row].cpu(), order), row
        want = (z[row].double() - z[row].double().logsumexp(0))[order]
        # fp32 sums and logs of values below 2^5
        assert (got[3][row].cpu().double() - want).abs().max() < 2.0**-16, row


def test_threads_do_not_share_workspaces(cuda):
    """Three threads with a stream each on rows of several parts."""
    announce("logit rows threads")
    bad = _bad(cuda)
    zs = [torch.randn(6, 140000, generator=torch.Generator().manual_seed(i)).half().to(cuda) for i in range(3)]
    t = torch.arange(6, device=cuda)
    want = [K.token_logprobs_fwd(z, t, 40, bad) for z in zs]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(cuda)):
                for _ in range(10):
                    got[i] = K.token_logprobs_fwd(zs[i], t, 40, bad)
                torch.cuda.current_stream(cuda).synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not errors, errors
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
