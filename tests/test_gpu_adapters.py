"""GPU parity of projections with low-rank adapters of many tasks against the
oracle in 64 bits on the same operands.  The tolerances are the oracle's: fp32 sums
32 deep, x A^T and dy B rounded to 16 bits (half a step: bf16 2^-8 of the value at
most, fp16 2^-11; in fp16 the largest of a tile's values stands at 2^13 to 2^14, so
the smallest are off by up to 2^-25 of 2^13: 2^-38 of it), and one rounding of the
results."""

import threading

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.model.functional import AdapterLinearFn, LinearFn
from eth_amd.packed import AdapterRows
from oracle.adapters import adapter_linear
from tests.conftest import announce

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0**-37}
TYPES = [torch.bfloat16, torch.float16]


def _rows(cuda, lens, ids, tail=0, scales=None):
    scales = [1.0 + 0.25 * (i % 5) for i in range(len(lens))] if scales is None else scales
    total = sum(lens) + tail
    counts = torch.tensor([*lens, tail])
    of_row = torch.tensor([*ids, -1]).repeat_interleave(counts).to(cuda)
    scale = torch.tensor([*scales, 1.0]).repeat_interleave(counts).to(cuda)
    return AdapterRows(lens, ids, scales, total, cuda), of_row, scale


def _operands(cuda, rows, k, n, r, adapters, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    o = dict(x=randn(rows, k), w=randn(n, k) / k**0.5, bias=randn(n) * 0.1, a=randn(adapters, r, k) / k**0.5,
             b=randn(adapters, n, r) / r**0.5, dy=randn(rows, n))
    return {name: t.to(dtype).to(cuda) for name, t in o.items()}


def _within(got, r, name):
    off, bound = (got.double() - r[name]).abs(), r["bound_" + name]
    assert not got.isnan().any() and not (off > bound).any(), (
        f"{name}: {off.max():.3e} off, {(off / bound).nan_to_num(0.0).max():.2f} of the bound")


def _run(o, rows, bias=True):
    y, saved = K.adapter_linear_fwd(o["x"], o["w"], o["bias"] if bias else None, o["a"], o["b"], rows, save=True)
    da, db = torch.full_like(o["a"], 3.0), torch.full_like(o["b"], 3.0)
    dx = K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, saved, True, (da, False), (db, False))
    return y, dx, da, db, saved


def _check(o, of_row, scale, got, bias=True):
    dt = o["x"].dtype
    r = adapter_linear(o["x"], o["w"], o["bias"] if bias else None, o["a"], o["b"], of_row, scale, o["dy"], HALF_STEP[dt],
                       LEAST[dt], FLOOR[dt])
    for name, t in zip(("y", "dx", "da", "db"), got):
        _within(t, r, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,ids,tail,adapters,k,n,r", [
    ([1], [0], 0, 1, 8, 8, 8), ([1, 1, 1], [2, 0, 2], 0, 3, 64, 40, 16), ([7, 1, 0, 5], [1, 0, -1, 1], 3, 4, 64, 72, 24),
    ([16, 17, 31, 32, 33], [0, 1, 0, 1, 0], 0, 2, 136, 264, 40), ([100, 3, 70], [-1, 5, 0], 40, 6, 520, 200, 64),
    ([1] * 40, [(7 * i) % 11 for i in range(40)], 0, 11, 256, 512, 8), ([300, 45], [0, 0], 1, 1, 72, 1032, 128),
    ([70, 33, 129, 5], [1, 0, -1, 1], 3, 3, 264, 520, 96), ([500, 20, 700], [1, 2, 1], 5, 3, 1000, 1048, 128),
    # the wide tiles, whole and with short ends; the depth in splits
    ([900, 1100, 700, 1400], [0, 1, 0, 2], 19, 3, 320, 2056, 16), ([2048, 2300], [1, 0], 0, 2, 128, 2048, 64),
    ([400, 120], [0, 1], 0, 2, 8192, 512, 32), ([130, 390], [1, 0], 0, 2, 512, 8192, 16),
    # two tiles a workgroup: of one adapter, of two, an odd last one; in pieces of the depth too
    ([2000, 33, 1, 2050, 64], [0, 1, 0, 2, 1], 3, 3, 64, 72, 40), ([4090, 17, 3], [1, 0, 2], 0, 3, 2056, 264, 128),
])
def test_forward_and_backward(cuda, dtype, lens, ids, tail, adapters, k, n, r):
    announce(f"adapters {dtype} lens={lens} ids={ids} tail={tail} k={k} n={n} r={r}")
    rows, of_row, scale = _rows(cuda, lens, ids, tail)
    o = _operands(cuda, rows.total, k, n, r, adapters, dtype, k + n + r)
    *got, saved = _run(o, rows)
    torch.cuda.synchronize()
    _check(o, of_row, scale, got)
    # again, and each gradient alone: the same bits
    *again, _ = _run(o, rows)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    plain, none = K.adapter_linear_fwd(o["x"], o["w"], o["bias"], o["a"], o["b"], rows)
    assert none is None and torch.equal(plain, got[0])
    dx = K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows)
    da, db = torch.empty_like(o["a"]), torch.empty_like(o["b"])
    assert K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, None, False, (da, False)) is None
    K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, saved, False, None, (db, False))
    assert torch.equal(dx, got[1]) and torch.equal(da, got[2]) and torch.equal(db, got[3])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_no_adapter(cuda, dtype):
    """They are the shared projection's, bit for bit; adapters without rows get
    zero gradients, or keep what they are added to."""
    announce(f"rows of no adapter {dtype}")
    for lens, ids in (([20, 30], [-1, -1]), ([0, 50], [0, -1])):
        rows, of_row, scale = _rows(cuda, lens, ids, 2)
        o = _operands(cuda, 52, 128, 256, 16, 2, dtype)
        *got, _ = _run(o, rows)
        assert torch.equal(got[0], K.gemm(o["x"], o["w"].t(), bias=o["bias"]))
        assert torch.equal(got[1], K.gemm(o["dy"], o["w"]))
        assert (got[2] == 0).all() and (got[3] == 0).all()
        kept = torch.full(o["a"].shape, 2.0, device=cuda)
        K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, None, False, (kept, True))
        assert (kept == 2.0).all()
    rows, of_row, scale = _rows(cuda, [40, 24], [-1, 0])
    o = _operands(cuda, 64, 128, 256, 16, 2, dtype)
    *got, _ = _run(o, rows, bias=False)
    assert torch.equal(got[0][:40], K.gemm(o["x"], o["w"].t())[:40]) and (got[2][1] == 0).all()
    _check(o, of_row, scale, got, bias=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_tasks_stay_apart(cuda, dtype):
    """Values that are not finite, in rows or adapters, reach no other task."""
    announce(f"adapters stay apart {dtype}")
    lens, ids = [37, 20, 50, 9], [0, 1, -1, 2]
    rows, *_ = _rows(cuda, lens, ids)
    o = _operands(cuda, 116, 128, 192, 32, 4, dtype)
    want = _run(o, rows)
    bad = {k: v.clone() for k, v in o.items()}
    bad["x"][37 + 4, 3], bad["dy"][60:90, 0], bad["a"][1, 0, 0] = float("nan"), float("inf"), float("nan")
    bad["a"][3], bad["b"][3] = float("nan"), float("inf")  # (of no rows)
    got = _run(bad, rows)
    fine = list(range(37)) + list(range(107, 116))
    for i in (0, 1):
        assert torch.equal(got[i][fine], want[i][fine])
    # rows of no adapter are their own
    assert torch.equal(got[0][57:107], want[0][57:107])
    for i in (2, 3):
        assert torch.equal(got[i][[0, 2, 3]], want[i][[0, 2, 3]])
    assert got[2][1].isnan().any()


def test_small_gradients_and_adapters_keep_their_digits(cuda):
    """In fp16, dy and adapters times powers of two give the gradients times
    them, bit for bit."""
    announce("small gradients of fp16 adapters")
    rows, of_row, scale = _rows(cuda, [40, 24, 70], [1, 0, 1], scales=[1.0, 0.5, 2.0])
    o = _operands(cuda, 134, 128, 192, 16, 2, torch.float16)
    o["dy"] = torch.where(o["dy"].abs() < 0.125, 0.5, o["dy"])
    o["b"] = torch.where(o["b"].abs() < 0.0625, 0.25, o["b"])

    def grads(o):
        _, saved = K.adapter_linear_fwd(o["x"], o["w"], None, o["a"], o["b"], rows, save=True)
        da, db = torch.empty(o["a"].shape, device=cuda), torch.empty(o["b"].shape, device=cuda)
        K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, saved, False, (da, False), (db, False))
        return da, db

    da, db = grads(o)
    small = dict(o, dy=o["dy"] * 2.0**-10, b=o["b"] * 2.0**-9)
    da2, db2 = grads(small)
    assert torch.equal(da2, da * 2.0**-19) and torch.equal(db2, db * 2.0**-10)
    tiny = dict(o, a=torch.where(o["a"].abs() < 2.0**-6, 2.0**-6, o["a"].float()).half() * 2.0**-8)
    big = dict(o, a=tiny["a"] * 2.0**8)
    assert torch.equal(grads(tiny)[1], grads(big)[1] * 2.0**-8)
    r = adapter_linear(small["x"], small["w"], None, small["a"], small["b"], of_row, scale, small["dy"], 2.0**-11, 2.0**-126,
                       2.0**-37)
    _within(da2, r, "da")
    _within(db2, r, "db")


def test_autograd_strides_and_main_grads(cuda):
    announce("adapters autograd, strides, main grads")
    lens, ids = [37, 0, 20, 7], [1, 0, 2, 1]
    rows, of_row, scale = _rows(cuda, lens, ids, 1)
    o = _operands(cuda, 65, 128, 192, 16, 3, torch.bfloat16)
    y, dx, da, db, _ = _run(o, rows)

    def leaves(**other):
        return {k: v.detach().clone().requires_grad_(True) for k, v in (o | other).items() if k != "dy"}

    def apply(v):
        return AdapterLinearFn.apply(v["x"], v["w"], v["bias"], v["a"], v["b"], rows)

    v = leaves()
    out = apply(v)
    got = torch.autograd.grad(out, [v[k] for k in ("x", "a", "b", "w", "bias")], o["dy"])
    for a, b in zip((out.detach(), *got[:3]), (y, dx, da, db)):
        assert torch.equal(a, b)
    # the shared weight's and bias's gradients are LinearFn's: of rows padded to a multiple of 8
    lin = {k: o[k].detach().clone().requires_grad_(True) for k in ("w", "bias")}
    pad = torch.nn.functional.pad
    ref = torch.autograd.grad(LinearFn.apply(pad(o["x"], (0, 0, 0, 7)), lin["w"], lin["bias"]), [lin["w"], lin["bias"]],
                              pad(o["dy"], (0, 0, 0, 7)))
    assert torch.equal(got[3], ref[0])
    assert (got[4].double() - o["dy"].double().sum(0)).abs().max() < 2.0**-8 * 40
    with torch.autograd.graph.save_on_cpu():
        v = leaves()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(apply(v), [v[k] for k in ("x", "a", "b")], o["dy"]),
                                                     (dx, da, db)))
    # strides, offsets, a leading shape, an expanded gradient, frozen parts
    wide_w = torch.full((192, 144), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide_w[:, 8:136] = o["w"]
    wide = torch.full((65, 152), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:, 16:144] = o["x"]
    shifted = torch.empty(65 * 128 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(65, 128).copy_(o["x"])
    for x in (wide[:, 16:144], shifted, o["x"].view(5, 13, 128), o["x"].t().contiguous().t()):
        leaf = x.detach().requires_grad_(True)
        out = AdapterLinearFn.apply(leaf, wide_w[:, 8:136], o["bias"], o["a"], o["b"], rows)
        assert torch.equal(out.reshape(65, 192), y) and out.shape[:-1] == x.shape[:-1]
        (g,) = torch.autograd.grad(out, leaf, o["dy"].view(out.shape))
        assert torch.equal(g.reshape(65, 128), dx) and g.shape == x.shape
    v = leaves()
    (ones,) = torch.autograd.grad(apply(v).sum(), v["a"])
    want = torch.empty_like(da)
    K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], torch.ones_like(o["dy"]), rows, None, False, (want, False))
    assert torch.equal(ones, want)
    # main grads: added, or stored where stale
    p = {k: torch.nn.Parameter(o[k].clone()) for k in ("w", "bias", "a", "b")}
    for t in p.values():
        t.main_grad = torch.ones(t.shape, device=cuda)
    p["a"]._eth_main_grad_stale = True
    fa, fb = torch.empty(o["a"].shape, device=cuda), torch.empty(o["b"].shape, device=cuda)
    saved = K.adapter_linear_fwd(o["x"], o["w"], None, o["a"], o["b"], rows, save=True)[1]
    K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, saved, False, (fa, False), (fb, False))
    AdapterLinearFn.apply(o["x"], p["w"], p["bias"], p["a"], p["b"], rows).backward(o["dy"])
    assert all(t.grad is None for t in p.values())
    assert torch.equal(p["a"].main_grad, fa) and torch.equal(p["b"].main_grad, 1.0 + fb)
    dw = o["dy"].double().t() @ o["x"].double()
    assert (p["w"].main_grad.double() - 1.0 - dw).abs().max() < 2.0**-14


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,k,n,r", [([1], 64, 72, 8), ([16, 3, 1], 264, 128, 16), ([5, 16], 2048, 512, 64),
                                        ([2, 9], 128, 1032, 128)])
def test_few_rows_keep_more_of_their_products(cuda, dtype, lens, k, n, r):
    """Segments of up to 16 rows: x A^T and dy B are held in two parts for dA and dB,
    off by half a step of what half a step left, the square of one rounding."""
    announce(f"adapters few rows {dtype} {lens} {k} {n} {r}")
    rows, of_row, scale = _rows(cuda, lens, list(range(len(lens))), 2)
    o = _operands(cuda, sum(lens) + 2, k, n, r, len(lens), dtype)
    saved = K.adapter_linear_fwd(o["x"], o["w"], None, o["a"], o["b"], rows, save=True)[1]
    da, db = torch.empty(o["a"].shape, device=cuda), torch.empty(o["b"].shape, device=cuda)
    K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, saved, False, (da, False), (db, False))
    r = adapter_linear(o["x"], o["w"], None, o["a"], o["b"], of_row, scale, o["dy"], HALF_STEP[dtype] ** 2, LEAST[dtype],
                       FLOOR[dtype])
    _within(da, r, "da")
    _within(db, r, "db")


def test_main_grads_anywhere(cuda):
    """Main grads that start anywhere in a buffer, and one parameter in both places."""
    announce("adapters main grads anywhere")
    rows, *_ = _rows(cuda, [50, 30], [1, 0], 3)
    o = _operands(cuda, 83, 64, 64, 64, 2, torch.bfloat16)
    fa, fb = torch.empty(o["a"].shape, device=cuda), torch.empty(o["b"].shape, device=cuda)
    saved = K.adapter_linear_fwd(o["x"], o["w"], None, o["a"], o["b"], rows, save=True)[1]
    K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["b"], o["dy"], rows, saved, False, (fa, False), (fb, False))
    p = {k: torch.nn.Parameter(o[k].clone()) for k in ("a", "b")}
    buffer = torch.ones(2 + 2 * fa.numel(), device=cuda)
    p["a"].main_grad, p["b"].main_grad = buffer[2:].view(2, *fa.shape)
    p["b"]._eth_main_grad_stale = True
    for times in (1.0, 2.0):
        AdapterLinearFn.apply(o["x"], o["w"], None, p["a"], p["b"], rows).backward(o["dy"])
        assert torch.equal(p["a"].main_grad, 1.0 + fa if times == 1 else 1.0 + fa + fa)
        assert torch.equal(p["b"].main_grad, times * fb) and (buffer[:2] == 1).all()
    both = torch.nn.Parameter(o["a"].clone())
    saved = K.adapter_linear_fwd(o["x"], o["w"], None, o["a"], o["a"], rows, save=True)[1]
    K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["a"], o["dy"], rows, saved, False, (fa, False), (fb, False))
    both.main_grad = buffer[2 : 2 + fa.numel()].view(fa.shape)
    both._eth_main_grad_stale = True
    AdapterLinearFn.apply(o["x"], o["w"], None, both, both, rows).backward(o["dy"])
    assert both.grad is None and torch.equal(both.main_grad, fa + fb)
    with pytest.raises(ValueError):
        K.adapter_linear_bwd(o["x"], o["w"], o["a"], o["a"], o["dy"], rows, saved, False, (fa, False), (fa, False))


def test_streams_threads_and_replays(cuda):
    announce("adapters streams, threads, graphs")
    lens, ids = [60, 3, 41], [0, 1, 0]
    rows, *_ = _rows(cuda, lens, ids)
    sets = [_operands(cuda, 104, 256, 320, 32, 2, torch.float16, s) for s in range(3)]
    for s in sets[1:]:
        for k in ("w", "bias", "a", "b"):
            s[k] = sets[0][k]

    def step(o):
        v = {k: o[k].detach().requires_grad_(True) for k in ("x", "a", "b")}
        y = AdapterLinearFn.apply(v["x"], o["w"], o["bias"], v["a"], v["b"], rows)
        return y.detach(), *torch.autograd.grad(y, [v["x"], v["a"], v["b"]], o["dy"])

    want = [step(o) for o in sets]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(step(s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    out = [None] * 2

    def work(i):
        for _ in range(4):
            out[i] = step(sets[i])
        torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, b in zip(out, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    held = {k: v.clone() for k, v in sets[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step(held)))
    for s in (0, 1, 2, 0):
        for k in held:
            held[k].copy_(sets[s][k])
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want[s]))
        step(sets[(s + 1) % 3])


def test_refusals(cuda):
    announce("adapter refusals")
    rows, *_ = _rows(cuda, [10, 6], [0, 2])
    o = _operands(cuda, 16, 64, 72, 16, 3, torch.bfloat16)
    good = dict(x2d=o["x"], weight=o["w"], bias=o["bias"], lora_a=o["a"], lora_b=o["b"], rows=rows)
    two = _rows(cuda, [10, 5], [0, 2])[0]
    flat = torch.zeros(16 * 64 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(16, 64)
    for change in (dict(x2d=o["x"].float()), dict(x2d=o["x"][:15]), dict(weight=o["w"].half()), dict(rows=two),
                   dict(lora_a=o["a"][:2], lora_b=o["b"][:2]), dict(lora_a=o["a"][:, :8]), dict(lora_b=o["b"][:2]),
                   dict(lora_a=o["a"][:, :12].contiguous(), lora_b=o["b"][:, :, :12].contiguous()),
                   dict(x2d=o["x"][:, :60].contiguous(), weight=o["w"][:, :60].contiguous(),
                        lora_a=o["a"][:, :, :60].contiguous()), dict(lora_a=o["a"].transpose(1, 2).contiguous().transpose(1, 2)),
                   dict(x2d=flat), dict(x2d=o["x"].t().contiguous().t()), dict(x2d=o["x"][:1].expand(16, 64)),
                   dict(bias=o["bias"][:64]), dict(bias=o["bias"].float()), dict(weight=o["w"].cpu()), dict(x2d=o["x"].cpu()),
                   dict(bias=o["bias"].cpu()), dict(x2d=o["x"].view(4, 4, 64))):
        with pytest.raises(ValueError):
            K.adapter_linear_fwd(**(good | change))
    saved = K.adapter_linear_fwd(**good, save=True)[1]
    da, db = torch.empty_like(o["a"]), torch.empty_like(o["b"])
    args = (o["x"], o["w"], o["a"], o["b"])
    for dy, kw in ((o["dy"].float(), {}), (o["dy"][:15], {}), (o["dy"].t().contiguous().t(), {}),
                   (o["dy"], dict(da=(da[:2], False))), (o["dy"], dict(da=(da, True))), (o["dy"], dict(db=(db, False))),
                   (o["dy"], dict(saved=(saved[0][:1], saved[1]), db=(db, False))),
                   (o["dy"], dict(saved=(saved[0], saved[1].double()), db=(db, False))), (o["dy"].cpu(), {})):
        with pytest.raises(ValueError):
            K.adapter_linear_bwd(*args, dy, rows, **kw)
