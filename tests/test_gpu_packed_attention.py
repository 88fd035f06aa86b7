"""GPU parity of packed causal attention with shared heads against the oracle
in 64 bits on the same 16-bit inputs.

Tolerances: the oracle gives, element by element, what roundings of half a
step (u = 2^-8 in bf16, 2^-11 in fp16) of P, of dS and of the stored results
can change.  Scores, exponentials and sums are fp32: scores of at most 128
products below 2^5 are off by 128 * 2^-24 * 2^5 = 2^-12 in the exponent at the
most, which changes P, and all that follows, by the same share: an eighth of u
in bf16, and as much as half of u in fp16, whose bound is doubled for it."""

import math
import threading

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.model.functional import PackedCausalAttentionFn
from eth_amd.packed import PackedSequences
from oracle.packed import packed_attention
from tests.conftest import announce

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
SLACK = {torch.bfloat16: 1.25, torch.float16: 2.0}


def _inputs(rows, n, m, hn, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    mixed = torch.randn(rows, n + 2 * m, hn, generator=gen).to(dtype)
    dout = torch.randn(rows, n * hn, generator=gen).to(dtype)
    return mixed, dout


def _split(mixed, n, m):
    return torch.split(mixed, (n, m, m), dim=1)


def _run(q, k, v, packed, dout, scale=None):
    out, lse = K.packed_attention_fwd(q, k, v, packed, scale)
    dq, dk, dv = (torch.full(t.shape, math.nan, dtype=t.dtype, device=t.device) for t in (q, k, v))
    K.packed_attention_bwd(q, k, v, out, dout, lse, packed, dq, dk, dv, scale)
    return dict(out=out.view(q.shape), lse=lse, dq=dq, dk=dk, dv=dv)


def _check(got, ref, dtype):
    for name in ("out", "dq", "dk", "dv"):
        g, r = got[name].double().cpu(), ref[name]
        off = (g - r).abs()
        bound = SLACK[dtype] * ref["bound_" + name] + 2.0**-22  # (and sums of values that cancel)
        if dtype == torch.float16:
            bound = bound + 2.0**-24  # half the smallest fp16 step
        assert not (off > bound).any() and not g.isnan().any(), (
            f"{name}: {off.max():.3e} off, {(off / bound).max():.2f} of the bound")
    lse = got["lse"].double().cpu() * math.log(2.0)
    real = ref["lse"].isfinite()
    assert torch.equal(lse.isfinite(), real)
    assert (lse - ref["lse"])[real].abs().max().item() < 2.0**-12 if real.any() else True


CASES = [
    # lengths, tail, n, m, hn
    ([1], 0, 1, 1, 64),
    ([1, 2, 0, 3], 0, 4, 2, 64),
    ([31, 32, 33], 5, 4, 1, 64),
    ([63, 64, 65, 0], 1, 2, 2, 128),
    ([127, 128, 129], 130, 6, 2, 96),
    ([300, 1, 200], 0, 8, 2, 80),
    ([513], 0, 3, 1, 40),
    ([640, 70], 0, 2, 1, 128),
    ([257, 19], 3, 8, 1, 8),
    ([0, 0, 5, 0], 200, 12, 6, 120),
    ([0, 0], 70, 4, 2, 128),  # no sequence at all
    ([], 3, 2, 2, 64),
    ([97] * 7, 0, 12, 12, 16),
    ([1025], 7, 4, 1, 128),
    ([1100, 40], 0, 2, 2, 72),
    # chains split over several workgroups, in every kernel
    ([1700, 33], 9, 2, 1, 64),
    ([5, 1650], 0, 2, 1, 80),
    ([1500], 0, 3, 1, 128),
    ([1345, 1281, 0, 600], 0, 4, 4, 128),
]


def test_cases_split_chains(cuda):
    """The cases meant to split do, and others do not."""
    splits = [PackedSequences(lengths, total=sum(lengths) + tail, device=cuda).plan(n, m, hn)[4:]
              for lengths, tail, n, m, hn in CASES]
    assert all(q[0] and k[0] for q, k in splits[-4:]) and not any(q[0] or k[0] for q, k in splits[:5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,tail,n,m,hn", CASES)
def test_forward_and_gradients(cuda, dtype, lengths, tail, n, m, hn):
    announce(f"packed attention {dtype} {lengths} +{tail} n={n} m={m} hn={hn}")
    rows = sum(lengths) + tail
    mixed, dout = _inputs(rows, n, m, hn, dtype, rows + n + hn)
    ref = packed_attention(*(t.double() for t in _split(mixed, n, m)), lengths, dout=dout.double().view(rows, n, hn),
                           u=U[dtype])
    got = _run(*_split(mixed.to(cuda), n, m), PackedSequences(lengths, total=rows, device=cuda), dout.to(cuda))
    torch.cuda.synchronize()
    _check(got, ref, dtype)


@pytest.mark.parametrize("scale", [0.02, 0.4])
def test_scale(cuda, scale):
    announce(f"packed attention scale {scale}")
    lengths, n, m, hn, dtype = [70, 131], 4, 2, 64, torch.bfloat16
    mixed, dout = _inputs(201, n, m, hn, dtype, 5)
    ref = packed_attention(*(t.double() for t in _split(mixed, n, m)), lengths, scale,
                           dout.double().view(201, n, hn), u=U[dtype])
    got = _run(*_split(mixed.to(cuda), n, m), PackedSequences(lengths, device=cuda), dout.to(cuda), scale)
    _check(got, ref, dtype)


@pytest.mark.parametrize("n,m,hn", [(4, 1, 64), (2, 2, 96), (4, 2, 128)])
def test_neighbours_do_not_meet(cuda, n, m, hn):
    """Non-finite values in one sequence and in the rows behind the last: the
    other sequences' outputs and gradients are the bits of clean inputs."""
    announce(f"packed attention non-finite neighbours n={n} m={m} hn={hn}")
    lengths, rows, dtype = [45, 70, 129, 33], 300, torch.bfloat16
    mixed, dout = _inputs(rows, n, m, hn, dtype, 11)
    packed = PackedSequences(lengths, total=rows, device=cuda)
    clean = _run(*_split(mixed.to(cuda), n, m), packed, dout.to(cuda))
    bad, dbad = mixed.clone(), dout.clone()
    for s in (slice(45, 115), slice(277, 300)):
        bad[s] = torch.tensor([math.inf, -math.inf, math.nan], dtype=dtype)[torch.arange(hn) % 3]
        dbad[s] = math.nan
    got = _run(*_split(bad.to(cuda), n, m), packed, dbad.to(cuda))
    keep = torch.ones(rows, dtype=torch.bool)
    keep[45:115] = False
    for name in ("out", "dq", "dk", "dv"):
        assert torch.equal(got[name][keep.to(cuda)], clean[name][keep.to(cuda)]), name
        assert (got[name][277:] == 0).all(), name


def test_layouts_and_broadcast_heads(cuda):
    """Head-major and broadcast inputs, and gradients written into views, give
    the bits of the contiguous call."""
    announce("packed attention layouts")
    lengths, n, m, hn, dtype = [100, 60], 4, 2, 64, torch.float16
    mixed, dout = _inputs(160, n, m, hn, dtype, 3)
    q, k, v = (t.contiguous().to(cuda) for t in _split(mixed, n, m))
    k = k[:, :1].expand(160, m, hn)
    packed = PackedSequences(lengths, device=cuda)
    dout = dout.to(cuda)
    want = _run(q, k.contiguous(), v, packed, dout)
    hq, hv = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, v))
    out, lse = K.packed_attention_fwd(hq, k, hv, packed)
    grads = torch.full((160, 2 * (n + 2 * m), hn), 7.0, dtype=dtype, device=cuda)
    dq, dk, dv = torch.split(grads[:, ::2], (n, m, m), dim=1)
    K.packed_attention_bwd(hq, k, hv, out, dout, lse, packed, dq, dk, dv)
    for name, g in (("out", out.view(q.shape)), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert torch.equal(g, want[name]), name
    assert (grads[:, 1::2] == 7.0).all()


def test_gradients_of_broadcast_inputs(cuda):
    """One key/value head broadcast to all by expand, and one row of queries to
    all rows: autograd adds up the copies' gradients."""
    announce("packed attention broadcast inputs")
    lengths, n, hn = [40, 33], 4, 64
    gen = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn(*s, generator=gen).half().to(cuda).requires_grad_(True)
               for s in ((1, n, hn), (73, 1, hn), (73, 1, hn)))
    dout = torch.randn(73, n * hn, generator=gen).half().to(cuda)
    packed = PackedSequences(lengths, device=cuda)
    out = PackedCausalAttentionFn.apply(q.expand(73, n, hn), k.expand(73, n, hn), v.expand(73, n, hn), packed)
    got = torch.autograd.grad(out, (q, k, v), dout)
    full = [t.detach().expand(73, n, hn).contiguous() for t in (q, k, v)]
    each = _run(*full, packed, dout)
    assert torch.equal(out.view(73, n, hn), each["out"])
    for g, name, dim in zip(got, ("dq", "dk", "dv"), (0, 1, 1)):
        want = each[name].double().sum(dim, keepdim=True)
        # (each copy's gradient is the kernel's; their sum may round in fp16 at every addition)
        assert g.shape == want.shape
        bound = each[name].double().abs().sum(dim, keepdim=True) * 2.0**-10 + 2.0**-20
        assert ((g.double() - want).abs() <= bound).all(), name


def test_given_output_and_rows_of_no_sequence(cuda):
    announce("packed attention given output")
    mixed, _ = _inputs(50, 4, 4, 64, torch.bfloat16, 9)
    q, k, v = _split(mixed.to(cuda), 4, 4)
    packed = PackedSequences([20, 11], total=50, device=cuda)
    want, _ = K.packed_attention_fwd(q, k, v, packed)
    out = torch.full((50, 256), math.nan, dtype=torch.bfloat16, device=cuda)
    got, lse = K.packed_attention_fwd(q, k, v, packed, out=out)
    assert got is out and torch.equal(out, want)
    assert (out[31:] == 0).all() and (lse[:, 31:] == -math.inf).all()


def test_strided_rows_past_32_bits(cuda):
    """Rows 2 MiB apart: a sequence of 4.2 GiB, and the next one behind it."""
    announce("packed attention rows past 32 bits")
    lengths, n, m, hn, dtype = [2100, 70], 2, 1, 64, torch.bfloat16
    rows = sum(lengths)
    mixed, dout = _inputs(rows, n, m, hn, dtype, 21)
    big = torch.empty(rows, 2**20, dtype=dtype, device=cuda)
    far = big[:, : (n + 2 * m) * hn].view(rows, n + 2 * m, hn)
    far.copy_(mixed)
    packed = PackedSequences(lengths, device=cuda)
    want = _run(*_split(mixed.to(cuda), n, m), packed, dout.to(cuda))
    got = _run(*_split(far, n, m), packed, dout.to(cuda))
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_autograd_streams_and_replays(cuda):
    """Through autograd, on another stream, in two streams at once, and captured
    into a graph that is replayed on new inputs between eager calls."""
    announce("packed attention autograd, streams, graphs")
    lengths, n, m, hn, dtype = [90, 1, 140], 4, 2, 128, torch.bfloat16
    rows = sum(lengths) + 6
    packed = PackedSequences(lengths, total=rows, device=cuda)
    sets = []
    for seed in range(3):
        mixed, dout = _inputs(rows, n, m, hn, dtype, seed)
        sets.append((mixed.to(cuda), dout.to(cuda)))

    def step(mixed, dout):
        leaf = mixed.detach().requires_grad_(True)
        out = PackedCausalAttentionFn.apply(*_split(leaf, n, m), packed)
        (grad,) = torch.autograd.grad(out, leaf, dout)
        return out.detach(), grad

    want = [step(*s) for s in sets]
    direct = _run(*_split(sets[0][0], n, m), packed, sets[0][1])
    assert torch.equal(want[0][0], direct["out"].view(rows, -1))
    assert torch.equal(want[0][1], torch.cat([direct[x] for x in ("dq", "dk", "dv")], 1))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(step(*s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))

    mixed, dout = (t.clone() for t in sets[0])

    def captured():
        q, k, v = _split(mixed, n, m)
        return _run(q, k, v, packed, dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = captured()
    for s, w in ((0, 0), (1, 1), (2, 2), (0, 0)):
        mixed.copy_(sets[s][0])
        dout.copy_(sets[s][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held["out"].view(rows, -1), want[w][0])
        assert torch.equal(torch.cat([held[x] for x in ("dq", "dk", "dv")], 1), want[w][1])
        step(*sets[(s + 1) % 3])


def test_equal_lengths_agree_with_the_batched_kernels(cuda):
    """Four sequences of 128 rows, equal heads: the same sums as the batched
    kernels' up to the order of fp32 additions, so equal up to one rounding of
    the output (2^-8 relative) where that order tips it."""
    announce("packed attention against batched")
    s, b, n, hn, dtype = 128, 4, 2, 64, torch.bfloat16
    mixed, _ = _inputs(s * b, n, n, hn, dtype, 8)
    q, k, v = _split(mixed.to(cuda), n, n)
    out, _ = K.packed_attention_fwd(q, k, v, PackedSequences([s] * b, device=cuda))
    q4, k4, v4 = (t.reshape(b, s, n, hn).transpose(0, 1) for t in (q, k, v))
    want, _ = K.attention_fwd(q4, k4, v4)
    want = want.transpose(0, 1).reshape(s * b, n * hn).float()
    off = (out.float() - want).abs()
    assert (off <= 2.0**-7 * want.abs() + 2.0**-14).all()


def test_refusals(cuda):
    announce("packed attention refusals")
    packed = PackedSequences([5, 3], device=cuda)
    bf16 = dict(dtype=torch.bfloat16, device=cuda)
    q, k = torch.zeros(8, 4, 64, **bf16), torch.zeros(8, 2, 64, **bf16)
    K.packed_attention_fwd(q, k, k, packed)
    bad = [
        (q[:7], k[:7], k[:7]),  # rows
        (q, k[:7], k[:7]),
        (q, k, k[:, :1]),  # v unlike k
        (q, torch.zeros(8, 3, 64, **bf16), torch.zeros(8, 3, 64, **bf16)),  # heads
        (q[..., :60], k[..., :60], k[..., :60]),  # head dim
        (q, k.half(), k.half()),  # types
        (q.float(), k.float(), k.float()),
        (q.cpu(), k.cpu(), k.cpu()),
        (q.view(8, 256), k, k),
        (torch.zeros(8, 4, 128, **bf16)[..., ::2], k, k),  # dim not contiguous
        (torch.zeros(8 * 256 + 8, **bf16)[4 : 4 + 8 * 256].view(8, 4, 64), k, k),  # alignment
        (torch.zeros(8, 260, **bf16)[:, :256].view(8, 4, 64), k, k),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            K.packed_attention_fwd(*args, packed)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            K.packed_attention_fwd(q, k, k, packed, scale)
    with pytest.raises(ValueError):
        K.packed_attention_fwd(q, k, k, packed, out=torch.zeros(8, 512, **bf16)[:, :256])
    out, lse = K.packed_attention_fwd(q, k, k, packed)
    good = dict(out=out, dout=out, lse=lse, dq=q.clone(), dk=k.clone(), dv=k.clone())

    def bwd(**changes):
        a = good | changes
        K.packed_attention_bwd(q, k, k, a["out"], a["dout"], a["lse"], packed, a["dq"], a["dk"], a["dv"])

    bwd()
    for changes in (dict(dout=out.view(8, 4, 64)), dict(lse=lse[:, :7]), dict(lse=lse.double()), dict(dk=q.clone()),
                    dict(dq=k.clone()), dict(dv=k[:, :1].expand(8, 2, 64)), dict(dq=q[:1].expand(8, 4, 64)),
                    dict(dout=torch.zeros(256, 8, **bf16).t())):
        with pytest.raises(ValueError):
            bwd(**changes)


def test_scale_of_a_tensor_is_its_value_of_the_call(cuda):
    announce("packed attention scale from a tensor")
    mixed, dout = _inputs(40, 4, 2, 64, torch.bfloat16, 31)
    packed = PackedSequences([25, 15], device=cuda)
    grads = []
    for scale in (0.25, torch.tensor(0.25), torch.tensor(0.25, device=cuda)):
        leaf = mixed.to(cuda).requires_grad_(True)
        out = PackedCausalAttentionFn.apply(*_split(leaf, 4, 2), packed, scale)
        if isinstance(scale, torch.Tensor):
            scale.fill_(3.0)
        grads.append(torch.autograd.grad(out, leaf, dout.to(cuda))[0])
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("dtype", U)
@pytest.mark.parametrize("hn", [64, 96, 128])
def test_scores_that_rise_and_fall_along_a_sequence(cuda, dtype, hn):
    """Whole numbers, whose products are exact: the scores of even queries rise
    by 46 (log2 units) every 64 keys, up to 370, and those of odd ones fall, so
    that the running maximum is taken again at every block or never.  An exponent
    is off by one rounding, 2^-24 * 2^9, and P by 2^-15 of itself."""
    announce(f"packed attention rising scores {dtype} hn={hn}")
    lengths, n, m = [520, 1, 40], 4, 2
    rows = sum(lengths)
    gen = torch.Generator().manual_seed(hn)
    mixed = torch.randint(-1, 2, (rows, n + 2 * m, hn), generator=gen).to(dtype)
    at = torch.arange(rows)
    mixed[:, :n, 0] = torch.where(at % 2 == 0, 8, -8).to(dtype)[:, None]
    mixed[:, n : n + m, 0] = (at // 2 % 256).to(dtype)[:, None]
    _, dout = _inputs(rows, n, m, hn, dtype, 3)
    scale = 0.125
    ref = packed_attention(*(t.double() for t in _split(mixed, n, m)), lengths, scale,
                           dout.double().view(rows, n, hn), u=U[dtype])
    got = _run(*_split(mixed.to(cuda), n, m), PackedSequences(lengths, device=cuda), dout.to(cuda), scale)
    _check(got, ref, dtype)


def test_a_query_of_nan_leaves_the_others(cuda):
    """NaN scores of one query make its wave take its maxima anew each block: the
    other rows are the clean call's but for their exponents' offsets (P rounded
    at another power of two: a step of bf16; lse, of at most 2^4, by 2^-20 a
    rounding)."""
    announce("packed attention NaN query")
    lengths, n, m, dtype = [200, 30], 4, 2, torch.bfloat16
    mixed, _ = _inputs(230, n, m, 64, dtype, 41)
    packed = PackedSequences(lengths, device=cuda)
    want, want_lse = K.packed_attention_fwd(*_split(mixed.to(cuda), n, m), packed)
    mixed[150, 1] = math.nan
    got, lse = K.packed_attention_fwd(*_split(mixed.to(cuda), n, m), packed)
    got, want = (t.view(230, n, 64) for t in (got, want))
    assert got[150, 1].isnan().all() and lse[1, 150].isnan()
    keep = torch.ones(230, n, dtype=torch.bool, device=cuda)
    keep[150, 1] = False
    assert torch.allclose(got[keep].float(), want[keep].float(), rtol=2.0**-7, atol=2.0**-9)
    assert torch.allclose(lse.t()[keep], want_lse.t()[keep], rtol=0, atol=2.0**-18)


@pytest.mark.parametrize("n,m,hn", [(4, 1, 64), (2, 2, 128)])
def test_very_many_sequences_of_one_row(cuda, n, m, hn):
    """A sequence of one row has P = 1: out is v, dq and dk are zero but for
    delta's rounding (dP - delta: the same products, summed in another order),
    dv the sum of dout over the group."""
    announce(f"packed attention 70000 sequences n={n} m={m} hn={hn}")
    rows, dtype = 70000, torch.bfloat16
    mixed, dout = _inputs(rows, n, m, hn, dtype, 51)
    # small whole numbers: every sum is exact
    dout = torch.randint(-2, 3, dout.shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    mixed[:, n + m :] = torch.randint(-2, 3, (rows, m, hn), generator=torch.Generator().manual_seed(2)).to(dtype)
    q, k, v = (t.contiguous().to(cuda) for t in _split(mixed, n, m))
    got = _run(q, k, v, PackedSequences([1] * rows, device=cuda), dout.to(cuda))
    do = dout.to(cuda).view(rows, n, hn)
    assert torch.equal(got["out"], v.repeat_interleave(n // m, 1))
    assert torch.equal(got["dv"], do.view(rows, m, n // m, hn).sum(2))
    assert (got["dq"] == 0).all() and (got["dk"] == 0).all()


def test_threads_share_a_plan(cuda):
    """Four threads with a stream each, forward and backward through one plan,
    its descriptors and splits made by whichever comes first."""
    announce("packed attention threads")
    lengths, n, m, hn, dtype = [1700, 33], 2, 1, 64, torch.bfloat16
    mixed, dout = _inputs(1733, n, m, hn, dtype, 61)
    args = [t.contiguous().to(cuda) for t in _split(mixed, n, m)]
    dout = dout.to(cuda)
    want = _run(*args, PackedSequences(lengths, device=cuda), dout)
    packed = PackedSequences(lengths, device=cuda)
    torch.cuda.synchronize()
    results, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(cuda)):
                for _ in range(5):
                    leaves = [t.clone().requires_grad_(True) for t in args]
                    out = PackedCausalAttentionFn.apply(*leaves, packed)
                    grads = torch.autograd.grad(out, leaves, dout)
                torch.cuda.current_stream(cuda).synchronize()
                results[i] = out.detach(), *grads
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for r in results:
        for g, name in zip(r, ("out", "dq", "dk", "dv")):
            assert torch.equal(g.view_as(want[name]), want[name]), name


def test_two_graphs_of_split_chains_replayed_in_turn(cuda):
    """Two captured training steps whose chains are split, their workspaces in
    one memory pool, replayed in turn on new inputs with eager calls between."""
    announce("packed attention two graphs, split chains")
    n, m, hn, dtype = 2, 1, 64, torch.bfloat16
    rows = 1733
    plans = [PackedSequences(x, device=cuda) for x in ([1700, 33], [20, 1713])]
    sets = [tuple(t.to(cuda) for t in _inputs(rows, n, m, hn, dtype, seed)) for seed in (71, 72, 73)]
    want = [[_run(*_split(x, n, m), p, do) for x, do in sets] for p in plans]
    buffers = [tuple(t.clone() for t in sets[0]) for _ in plans]
    graphs, held, pool = [], [], None
    for p, (x, do) in zip(plans, buffers):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _run(*_split(x, n, m), p, do)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            held.append(_run(*_split(x, n, m), p, do))
        pool = g.pool()
        graphs.append(g)
    for i in (0, 1, 2, 0):
        for g, h, w, (x, do), p in zip(graphs, held, want, buffers, plans):
            x.copy_(sets[i][0])
            do.copy_(sets[i][1])
            g.replay()
            eager = _run(*_split(sets[i - 1][0], n, m), p, sets[i - 1][1])
            torch.cuda.synchronize()
            for name in ("out", "lse", "dq", "dk", "dv"):
                assert torch.equal(h[name], w[i][name]), name
                assert torch.equal(eager[name], w[i - 1][name]), name
