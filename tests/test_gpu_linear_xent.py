"""GPU parity of the linear head's cross entropy without its logits against the
oracle in 64 bits on the same operands.  The tolerances are the oracle's: fp32
products summed 32 deep, exponentials and sums in fp32, dz rounded to 16 bits
(half a step: bf16 2^-8 of the value at most, fp16 2^-11; dz of fp16 carries 2^14,
so one below 2^-39 of its row's dloss is off by up to 2^-39), and one rounding of
the gradients."""

import threading

import pytest
import torch

from eth_amd import kernels as K
from eth_amd import _native as nat
from eth_amd.model.functional import CrossEntropyFn, LinearCrossEntropyFn, LinearFn, overlapped_wgrad
from oracle.linear_xent import linear_xent
from tests.conftest import announce

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
LEAST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25, torch.float32: 2.0**-126}
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0**-38}
TYPES = [torch.bfloat16, torch.float16]


def _operands(cuda, rows, H, V, dtype, seed=0, ignored=0.0, spread=2.0, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(V, H, generator=gen) * (spread / H**0.5)
    labels = torch.randint(0, V, (rows,), generator=gen)
    h = torch.randn(rows, H, generator=gen) + w[labels]
    labels[torch.randperm(rows, generator=gen)[: int(rows * ignored)]] = -100
    dloss = (torch.rand(rows, generator=gen) + 0.5) * size
    return h.to(dtype).to(cuda), w.to(dtype).to(cuda), labels.to(cuda), dloss.to(cuda)


def _bad(cuda):
    return torch.zeros(1, dtype=torch.int32, device=cuda)


def _within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert not got.isnan().any() and not (off > bound).any(), (
        f"{what}: {off.max():.3e} off, {(off / bound).nan_to_num(0.0).max():.2f} of the bound")


def _check(h, w, labels, loss, dloss, dh, dw, dw_type=None):
    dt = h.dtype
    r = linear_xent(h, w, labels, -100, dloss, HALF_STEP[dt], LEAST[dt], FLOOR[dt])
    _within(loss, r["loss"], r["bound_loss"], "loss")
    _within(dh, r["dh"], r["bound_dh"], "dh")
    _within(dw, r["dw"], r["bound_dw"], "dw")
    gone = (labels == -100) | (dloss == 0)
    assert (loss[labels == -100] == 0).all() and (dh[gone] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,H,V,ignored", [
    (1, 8, 1, 0.0), (1, 64, 2, 0.0), (2, 8, 7, 0.0), (3, 72, 129, 0.0), (16, 64, 256, 0.5), (17, 136, 1001, 0.3),
    (64, 128, 5000, 0.0), (65, 40, 4097, 0.1), (130, 256, 3001, 0.6), (300, 200, 2500, 0.0), (257, 1024, 513, 0.02),
    (1000, 64, 9000, 0.2), (700, 96, 20001, 0.0), (1, 16, 40001, 0.0), (37, 24, 30000, 0.1),
])
def test_loss_and_gradients(cuda, dtype, rows, H, V, ignored):
    announce(f"linear xent {dtype} rows={rows} H={H} V={V} ignored={ignored}")
    h, w, labels, dloss = _operands(cuda, rows, H, V, dtype, rows + V, ignored)
    bad = _bad(cuda)
    loss, lse = K.linear_xent_fwd(h, w, labels, bad)
    dh, dw = K.linear_xent_bwd(h, w, labels, lse, dloss)
    torch.cuda.synchronize()
    assert bad.item() == 0
    _check(h, w, labels, loss, dloss, dh, dw)
    again = K.linear_xent_bwd(h, w, labels, lse, dloss)
    assert torch.equal(dh, again[0]) and torch.equal(dw, again[1])
    one, _ = K.linear_xent_bwd(h, w, labels, lse, dloss, need_dweight=False)
    _, other = K.linear_xent_bwd(h, w, labels, lse, dloss, need_dhidden=False)
    assert torch.equal(dh, one) and torch.equal(dw, other)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,H,V,ignored", [(1, 64, 3001, 0.0), (5, 128, 1000, 0.4), (64, 200, 2504, 0.0)])
def test_few_rows_keep_more_of_dz(cuda, dtype, rows, H, V, ignored):
    """Up to 64 rows dz is held in two parts: off by half a step of what half a
    step left, the square of one rounding."""
    announce(f"linear xent few rows {dtype} rows={rows}")
    h, w, labels, dloss = _operands(cuda, rows, H, V, dtype, rows, ignored)
    _, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    dw = torch.empty(V, H, device=cuda)
    dh, _ = K.linear_xent_bwd(h, w, labels, lse, dloss, dweight=dw)
    r = linear_xent(h, w, labels, -100, dloss, HALF_STEP[dtype] ** 2, LEAST[dtype], FLOOR[dtype])
    _within(dh, r["dh"], r["bound_dh"] + 1.001 * HALF_STEP[dtype] * r["dh"].abs(), "dh")
    _within(dw, r["dw"], r["bound_dw"], "dw")
    # a row without a finite gradient reaches itself alone
    dloss[0] = float("inf")
    if labels[0] != -100:
        bad, _ = K.linear_xent_bwd(h, w, labels, lse, dloss, dweight=dw)
        assert torch.equal(bad[1:], dh[1:]) and not bad[0].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES)
def test_several_pieces_of_the_vocabulary(cuda, dtype):
    """32768 rows of 9001 logits: three pieces, the last of an odd width."""
    announce(f"linear xent in pieces {dtype}")
    h, w, labels, dloss = _operands(cuda, 32768, 16, 9001, dtype, 3, 0.25)
    loss, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    dh, dw = K.linear_xent_bwd(h, w, labels, lse, dloss)
    _check(h, w, labels, loss, dloss, dh, dw)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_and_weights_of_wider_buffers(cuda, dtype):
    announce(f"linear xent strides {dtype}")
    h, w, labels, dloss = _operands(cuda, 70, 64, 777, dtype, 5, 0.1)
    wide_h, wide_w = torch.full((70, 104), float("nan"), dtype=dtype, device=cuda), torch.full((777, 72), float("nan"), dtype=dtype, device=cuda)
    wide_h[:, 8:72], wide_w[:, :64] = h, w
    vh, vw = wide_h[:, 8:72], wide_w[:, :64]
    loss, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    loss2, lse2 = K.linear_xent_fwd(vh, vw, labels, _bad(cuda))
    assert torch.equal(loss, loss2)
    for a, b in zip(K.linear_xent_bwd(h, w, labels, lse, dloss), K.linear_xent_bwd(vh, vw, labels, lse2, dloss)):
        assert torch.equal(a, b)
    # rows that the kernels cannot read in place are copied by the autograd function
    odd = torch.cat([h, h[:, :3]], 1)[:, :64]
    shifted = torch.empty(70 * 64 + 1, dtype=dtype, device=cuda)[1:].view(70, 64).copy_(h)
    for x in (odd, shifted, h.t().contiguous().t(), h.view(7, 10, 64).transpose(0, 1)):
        leaf = x.detach().requires_grad_(True)
        lab = labels.view(7, 10).t() if x.dim() == 3 else labels
        out = LinearCrossEntropyFn.apply(leaf, w, lab, _bad(cuda))
        back = out.t().reshape(-1) if x.dim() == 3 else out
        assert torch.allclose(back, loss, rtol=1e-5, atol=1e-5) if x.dim() == 3 else torch.equal(back, loss)
        (dx,) = torch.autograd.grad(out.sum(), leaf)
        assert dx.shape == x.shape


def test_weights_and_gradients_beyond_two_gibibytes(cuda):
    """A head whose rows lie 64 KiB apart, 2.6 GB in all, and fp32 gradients of 2.3 GB."""
    announce("linear xent beyond 2 GiB")
    h, w, labels, dloss = _operands(cuda, 33, 64, 40000, torch.bfloat16, 21)
    labels[:3] = torch.tensor([39999, 32768, 32767])
    wide = torch.empty(40000, 32768, dtype=torch.bfloat16, device=cuda)[:, 8:72].copy_(w)
    loss, lse = K.linear_xent_fwd(h, wide, labels, _bad(cuda))
    dh, dw = K.linear_xent_bwd(h, wide, labels, lse, dloss)
    _check(h, w, labels, loss, dloss, dh, dw)
    del wide
    gen = torch.Generator(device=cuda).manual_seed(22)
    randn = lambda *s: torch.randn(*s, generator=gen, device=cuda).bfloat16()  # noqa: E731
    h, w, labels = randn(3, 4096), randn(140000, 4096) * 2.0**-6, torch.tensor([139999, 0, 131072], device=cuda)
    loss, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    dw = torch.ones(140000, 4096, device=cuda)
    dh, _ = K.linear_xent_bwd(h, w, labels, lse, dloss[:3], dweight=dw, accumulate=True)
    dw -= 1.0  # (exact but for the rounding of the sum, 2^-24 of at most 8)
    r = linear_xent(h, w, labels, -100, dloss[:3], HALF_STEP[torch.bfloat16], LEAST[torch.bfloat16])
    _within(dh, r["dh"], r["bound_dh"], "dh")
    _within(dw, r["dw"], r["bound_dw"] + 2.0**-21, "dw")


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_take_no_part(cuda, dtype):
    """What ignored rows, and backward rows without upstream gradient, hold
    reaches nothing; labels outside the vocabulary are clamped and flagged."""
    announce(f"linear xent rows that take no part {dtype}")
    h, w, labels, dloss = _operands(cuda, 40, 64, 300, dtype, 6, 0.3)
    dloss[labels == -100] = float("nan")
    dloss[::7] = 0.0
    poison = h.clone()
    poison[labels == -100] = torch.tensor(float("nan"), dtype=dtype)
    poison[int((labels == -100).nonzero()[0])] = float("inf")
    bad = _bad(cuda)
    loss, lse = K.linear_xent_fwd(poison, w, labels, bad)
    gone = poison.clone()
    gone[::7] = float("nan")  # (their losses are there; their rows are not read again)
    dh, dw = K.linear_xent_bwd(gone, w, labels, lse, dloss)
    assert bad.item() == 0
    clean = torch.where((labels == -100)[:, None], torch.zeros_like(h), h)
    _check(clean, w, labels, loss, torch.where(labels == -100, 0.0, dloss), dh, dw)
    # another value to ignore
    loss7, _ = K.linear_xent_fwd(poison, w, torch.where(labels == -100, 7, labels.masked_fill(labels == 7, 8)), bad, 7)
    assert (loss7[labels == -100] == 0).all() and bad.item() == 0
    wild = labels.clone()
    wild[:3] = torch.tensor([-1, 300, 2**40])
    loss, lse = K.linear_xent_fwd(clean, w, wild, bad)
    r = linear_xent(clean, w, wild)
    _within(loss, r["loss"], r["bound_loss"], "loss of clamped labels")
    assert bad.item() == 1
    # nothing scored
    none = torch.full_like(labels, -100)
    loss, lse = K.linear_xent_fwd(torch.full_like(h, float("nan")), w, none, _bad(cuda))
    for g in K.linear_xent_bwd(torch.full_like(h, float("nan")), w, none, lse, dloss):
        assert (g == 0).all()
    assert (loss == 0).all()


def test_values_that_are_not_finite(cuda):
    announce("linear xent non-finite values")
    h, w, labels, dloss = _operands(cuda, 20, 64, 400, torch.bfloat16, 7)
    h[3, 5], h[4, 0] = float("nan"), float("inf")
    loss, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    dh, _ = K.linear_xent_bwd(h, w, labels, lse, dloss)
    hurt = torch.zeros(20, dtype=torch.bool, device=cuda)
    hurt[3:5] = True
    assert loss[hurt].isnan().all() and loss[~hurt].isfinite().all()
    assert dh[hurt].isnan().any(1).all() and dh[~hurt].isfinite().all()
    # logits of thousands: one probability is 1, the rest 0
    h, w, labels, dloss = _operands(cuda, 20, 64, 400, torch.bfloat16, 8, spread=600.0)
    loss, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    dh, dw = K.linear_xent_bwd(h, w, labels, lse, dloss)
    _check(h, w, labels, loss, dloss, dh, dw)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_any_size_keep_their_digits(cuda, dtype):
    """Upstream gradients times a power of two give gradients times it, bit for
    bit, where the results do not leave the type's range."""
    announce(f"linear xent gradient sizes {dtype}")
    h, w, labels, dloss = _operands(cuda, 50, 64, 1000, dtype, 9)
    dloss[::5] *= 2.0**-9
    _, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    dw = torch.empty(1000, 64, device=cuda)
    K.linear_xent_bwd(h, w, labels, lse, dloss, need_dhidden=False, dweight=dw)
    for k in (-40, -13, 9, 40):
        other = torch.empty_like(dw)
        K.linear_xent_bwd(h, w, labels, lse, dloss * 2.0**k, need_dhidden=False, dweight=other)
        assert torch.equal(other, dw * 2.0**k)
    r = linear_xent(h, w, labels, -100, dloss, HALF_STEP[dtype], LEAST[torch.float32], FLOOR[dtype])
    _within(dw, r["dw"], r["bound_dw"], "fp32 dw")


@pytest.mark.parametrize("rows,H,V", [(33, 64, 500), (300, 512, 3000), (304, 512, 3000)])
def test_weight_gradients_into_main_grad(cuda, rows, H, V):
    """Added into an fp32 main_grad, or stored where it is stale; 16-bit
    gradients are returned; the same in a context of overlapped weight
    gradients whose weight LinearFn uses too."""
    announce(f"linear xent main grad rows={rows}")
    h, w, labels, dloss = _operands(cuda, rows, H, V, torch.bfloat16, 10, 0.1)
    w = torch.nn.Parameter(w)
    h.requires_grad_(True)
    _, lse = K.linear_xent_fwd(h, w, labels, _bad(cuda))
    want = torch.empty(V, H, device=cuda)
    K.linear_xent_bwd(h.detach(), w.detach(), labels, lse, dloss, dweight=want)

    def backward():
        LinearCrossEntropyFn.apply(h, w, labels, _bad(cuda)).backward(dloss)

    w.main_grad = torch.full((V, H), 3.0, device=cuda)
    backward()
    assert w.grad is None and torch.equal(w.main_grad, 3.0 + want)
    w._eth_main_grad_stale = True
    backward()
    assert torch.equal(w.main_grad, want)
    backward()
    assert torch.equal(w.main_grad, want + want)
    dy = torch.randn(rows, V // 8 * 8, device=cuda).bfloat16()
    if V % 8 == 0 and rows % 8 == 0:  # (what LinearFn takes)
        w.main_grad.zero_()
        x = h.detach().clone()
        LinearFn.apply(x, w, None).backward(dy)
        backward()
        LinearFn.apply(x, w, None).backward(dy)
        whole = w.main_grad.clone()
        for other in (None, torch.cuda.Stream()):
            w.main_grad.zero_()
            torch.cuda.synchronize()
            with overlapped_wgrad():
                LinearFn.apply(x, w, None).backward(dy)
                if other is None:
                    backward()
                else:
                    other.wait_stream(torch.cuda.current_stream())
                    with torch.cuda.stream(other):
                        backward()
                LinearFn.apply(x, w, None).backward(dy)
            torch.cuda.synchronize()
            assert torch.equal(w.main_grad, whole)
    # one that starts anywhere in its buffer
    buffer = torch.ones(V * H + 2, device=cuda)
    w.main_grad = buffer[2:].view(V, H)
    backward()
    assert w.grad is None and torch.equal(w.main_grad, 1.0 + want)
    w._eth_main_grad_stale = True
    backward()
    assert torch.equal(w.main_grad, want) and (buffer[:2] == 1).all()
    del w.main_grad
    backward()
    assert w.grad.dtype == torch.bfloat16
    _within(w.grad, want.double(), 1.001 * HALF_STEP[torch.bfloat16] * want.double().abs() + LEAST[torch.bfloat16], "grad")


def test_beside_the_head_and_loss_with_logits(cuda):
    """The framework's own pair, whose logits are rounded to 16 bits: z off by
    2^-8 |z|, so the loss by that of the label's and the largest logits."""
    announce("linear xent beside LinearFn and CrossEntropyFn")
    h, w, labels, dloss = _operands(cuda, 200, 256, 1000, torch.bfloat16, 11)
    bad = _bad(cuda)
    loss = LinearCrossEntropyFn.apply(h.view(4, 50, 256), w, labels.view(4, 50), bad)
    kept = CrossEntropyFn.apply(LinearFn.apply(h, w, None).view(4, 50, 1000), labels.view(4, 50), bad)
    top = (h.float() @ w.float().t()).abs().amax()
    assert loss.shape == (4, 50) and (loss - kept).abs().max() < 2 * 2.0**-8 * top


def test_streams_threads_and_replays(cuda):
    announce("linear xent streams, threads, graphs")
    sets = [_operands(cuda, 90, 64, 1000, torch.bfloat16, s, 0.2) for s in range(3)]
    w = sets[0][1]

    def step(h, labels, dloss):
        leaf, lw = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = LinearCrossEntropyFn.apply(leaf, lw, labels, _bad(cuda))
        return loss.detach(), *torch.autograd.grad(loss, (leaf, lw), dloss)

    pick = [(h, labels, dloss) for h, _, labels, dloss in sets]
    want = [step(*s) for s in pick]
    torch.cuda.synchronize()
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, b) for a, b in zip(step(*pick[0]), want[0]))
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for st, s in zip(streams, pick):
        with torch.cuda.stream(st):
            got.append(step(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    out = [None] * 2

    def work(i):
        for _ in range(4):
            out[i] = step(*pick[i])
        torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, b in zip(out, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    held, bad = [x.clone() for x in pick[0]], _bad(cuda)

    def captured():
        h, labels, dloss = held
        loss, lse = K.linear_xent_fwd(h, w, labels, bad)
        return loss, *K.linear_xent_bwd(h, w, labels, lse, dloss)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, captured()))
    for s in (0, 1, 2, 0):
        for a, b in zip(held, pick[s]):
            a.copy_(b)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want[s]))
        step(*pick[(s + 1) % 3])
    h = torch.zeros(0, 64, dtype=torch.bfloat16, device=cuda).requires_grad_(True)
    lw = w.detach().requires_grad_(True)
    empty = LinearCrossEntropyFn.apply(h, lw, torch.zeros(0, dtype=torch.int64, device=cuda), bad)
    dh, dw = torch.autograd.grad(empty.sum(), (h, lw))
    assert empty.shape == (0,) and dh.shape == (0, 64) and (dw == 0).all()


def test_refusals(cuda):
    announce("linear xent refusals")
    h, w, labels, dloss = _operands(cuda, 10, 64, 100, torch.bfloat16)
    bad = _bad(cuda)
    lse = torch.zeros(10, device=cuda)
    for args in ((h.float(), w.float(), labels, bad), (h, w.half(), labels, bad), (h[:, :56], w, labels, bad),
                 (h[:, :60].contiguous(), w[:, :60].contiguous(), labels, bad), (h, w, labels.int(), bad),
                 (h, w, labels[:9], bad), (h, w, labels, bad.float()), (h, w.t().contiguous().t(), labels, bad),
                 (h, w[:, 4:60], labels, bad), (h.cpu(), w.cpu(), labels.cpu(), bad.cpu()), (h, w.cpu(), labels, bad),
                 (h[:1].expand(10, 64), w, labels, bad), (h[0], w, labels, bad)):
        with pytest.raises(ValueError):
            K.linear_xent_fwd(*args)
    for kw in (dict(dweight=torch.zeros(100, 64, device=cuda).bfloat16()), dict(dweight=torch.zeros(99, 64, device=cuda)),
               dict(accumulate=True), dict(dweight=torch.zeros(6401, device=cuda)[1:].view(100, 64))):
        with pytest.raises(ValueError):
            K.linear_xent_bwd(h, w, labels, lse, dloss, **kw)
    for bad_lse, bad_g in ((lse[:9], dloss), (lse.double(), dloss), (lse, dloss.half()), (lse, dloss.cpu())):
        with pytest.raises(ValueError):
            K.linear_xent_bwd(h, w, labels, bad_lse, bad_g)
    with pytest.raises(ValueError):
        LinearCrossEntropyFn.apply(h, w, labels.view(2, 5), bad)
