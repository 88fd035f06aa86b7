"""GPU parity of the fused norms around a residual (post-norm, gate, scaled
residual, next norm) against the oracle in 64 bits on the same operands.  The
tolerances are the oracle's: fp32 sums whose depth follows from the kernels'
layout, and one rounding of half a step of each 16-bit result."""

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.model.functional import GatedResidualNormFn
from oracle import residual_norm as oracle
from tests.conftest import announce

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}
TYPES = [torch.bfloat16, torch.float16]
NAMES = ("dpost_gamma", "dpost_beta", "dgate", "dgamma", "dbeta")


def _operands(cuda, rows, cols, dtype, rms, gate, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    o = dict(x=randn(rows, cols) * 0.7 + 0.2, residual=randn(rows, cols) * 2 - 0.5, pg=1 + 0.2 * randn(cols),
             pb=None if rms else 0.1 * randn(cols), gate=0.5 + 0.3 * randn(cols) if gate else None,
             gamma=1 + 0.2 * randn(cols), beta=None if rms else 0.1 * randn(cols), dh=randn(rows, cols),
             dy=randn(rows, cols))
    return {k: None if v is None else v.to(dtype).to(cuda) for k, v in o.items()}


def _params(o):
    return o["pg"], o["pb"], o["gate"], o["gamma"], o["beta"]


def _forward(o, scale, eps, rms):
    return K.residual_norm_fwd(o["x"], o["residual"], o["pg"], o["pb"], o["gate"], scale, o["gamma"], o["beta"], eps, rms)


def _backward(o, stats, dh, dy, scale, eps, rms, grads, **kw):
    pg, pb, gate, gamma, beta = _params(o)
    return K.residual_norm_bwd(o["x"], o["residual"], stats, dh, dy, pg, pb, gate, scale, gamma, beta, eps, rms, grads, **kw)


def _grads(o, fp32=False):
    return [None if p is None else (torch.full_like(p, 7.0, dtype=torch.float32 if fp32 else p.dtype), False)
            for p in _params(o)]


def _within(got, r, name):
    off, bound = (got.double() - r[name]).abs(), r["bound_" + name]
    assert not got.isnan().any() and not (off > bound).any(), (
        f"{name}: {off.max():.3e} off, {(off / bound).nan_to_num(0.0).max():.2f} of the bound")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rms,gate,scale", [(False, True, 1.0), (False, False, 0.7), (True, True, -0.5), (True, False, 0.0)])
@pytest.mark.parametrize("rows,cols", [(1, 8), (2, 40), (3, 504), (17, 512), (5, 520), (9, 1024), (33, 1032), (7, 2048),
                                       (4, 2568), (21, 4096), (6, 4104), (3, 5120), (2, 8184), (11, 8192), (700, 264),
                                       (3001, 1032)])
def test_forward_and_backward(cuda, dtype, rms, gate, scale, rows, cols):
    announce(f"residual norm {dtype} rows={rows} cols={cols} rms={rms} gate={gate} scale={scale}")
    o = _operands(cuda, rows, cols, dtype, rms, gate, rows + cols)
    eps = 1e-5
    h, y, stats = _forward(o, scale, eps, rms)
    u, least = HALF_STEP[dtype], LEAST[dtype]
    r = oracle.forward(o["x"], o["residual"], o["pg"], o["pb"], o["gate"], scale, o["gamma"], o["beta"], eps, rms, u,
                       least)
    _within(h, r, "h")
    _within(y, r, "y")
    for dh, dy in ((o["dh"], o["dy"]), (o["dh"], None), (None, o["dy"])):
        grads = _grads(o)
        dx, dres = _backward(o, stats, dh, dy, scale, eps, rms, grads)
        r = oracle.backward(o["x"], o["residual"], dh, dy, o["pg"], o["pb"], o["gate"], scale, o["gamma"], eps, rms, u, least)
        _within(dx, r, "dx")
        _within(dres, r, "dresidual")
        for name, pair in zip(NAMES, grads):
            if pair is not None:
                _within(pair[0], r, name)
    # fp32 gradients, stored and added; nothing else asked for
    wide = _grads(o, fp32=True)
    nothing = _backward(o, stats, None, o["dy"], scale, eps, rms, wide, need_dx=False, need_dresidual=False)
    assert nothing == (None, None)
    r = oracle.backward(o["x"], o["residual"], None, o["dy"], o["pg"], o["pb"], o["gate"], scale, o["gamma"], eps, rms)
    once = [None if p is None else p[0].clone() for p in wide]
    for name, pair in zip(NAMES, wide):
        if pair is not None:
            _within(pair[0], r, name)
    more = [None if p is None else (p[0], True) for p in wide]
    _backward(o, stats, None, o["dy"], scale, eps, rms, more)
    for pair, one in zip(wide, once):
        assert pair is None or torch.equal(pair[0], one + one)


def test_rows_stay_apart(cuda):
    """What is not finite in one row reaches no other row's results."""
    announce("residual norm rows apart")
    for rms in (False, True):
        o = _operands(cuda, 12, 1032, torch.bfloat16, rms, True)
        clean = _forward(o, 0.7, 1e-5, rms)
        want = _backward(o, clean[2], o["dh"], o["dy"], 0.7, 1e-5, rms, _grads(o))
        bad = dict(o, x=o["x"].clone(), residual=o["residual"].clone(), dy=o["dy"].clone())
        bad["x"][2, 5], bad["residual"][4, 1000], bad["dy"][6, 0] = float("nan"), float("inf"), float("nan")
        h, y, stats = _forward(bad, 0.7, 1e-5, rms)
        fine = [i for i in range(12) if i not in (2, 4)]
        assert torch.equal(h[fine], clean[0][fine]) and torch.equal(y[fine], clean[1][fine])
        assert h[2].isnan().all() and y[4].isnan().any()
        got = _backward(bad, stats, o["dh"], bad["dy"], 0.7, 1e-5, rms, _grads(o))
        fine.remove(6)
        for a, b in zip(got, want):
            assert torch.equal(a[fine], b[fine])
        assert got[0][6].isnan().all()
    # rows of one value: a deviation of zero, kept finite by eps
    o = _operands(cuda, 3, 64, torch.float16, False, False)
    o["x"].fill_(2.5)
    o["residual"].fill_(-1.0)
    o["pb"].zero_()
    h, y, stats = _forward(o, 1.0, 1e-5, False)
    assert torch.equal(h, o["residual"]) and torch.equal(y, o["beta"].expand_as(y))
    dx, dres = _backward(o, stats, o["dh"], None, 1.0, 1e-5, False, _grads(o))
    assert dx.isfinite().all() and torch.equal(dres, o["dh"])


def test_rows_beyond_two_gibibytes(cuda):
    """The last rows of 2.3 GB tensors: those of a call with them alone."""
    announce("residual norm beyond 2 GiB")
    rows, cols = 140000, 8192
    gen = torch.Generator(device=cuda).manual_seed(3)
    few = _operands(cuda, 9, cols, torch.float16, False, True)
    big = {k: v if v is None or v.dim() == 1 else torch.randn(rows, cols, generator=gen, device=cuda, dtype=v.dtype)
           for k, v in few.items()}
    for k in ("x", "residual", "dh", "dy"):
        big[k][-9:] = few[k]
    h, y, stats = _forward(big, 0.7, 1e-5, False)
    want = _forward(few, 0.7, 1e-5, False)
    assert torch.equal(h[-9:], want[0]) and torch.equal(y[-9:], want[1]) and torch.equal(stats[:, -9:], want[2])
    got = _backward(big, stats, big["dh"], big["dy"], 0.7, 1e-5, False, [None] * 5)
    want = _backward(few, want[2], few["dh"], few["dy"], 0.7, 1e-5, False, [None] * 5)
    assert all(torch.equal(a[-9:], b) for a, b in zip(got, want))


def _leaves(o):
    return {k: None if v is None or k in ("dh", "dy") else v.detach().clone().requires_grad_(True) for k, v in o.items()}


def _apply(leaf, scale=0.7, rms=False):
    return GatedResidualNormFn.apply(leaf["x"], leaf["residual"], leaf["pg"], leaf["pb"], leaf["gate"], scale,
                                     leaf["gamma"], leaf["beta"], 1e-5, rms)


def test_autograd_main_grads_streams_and_replays(cuda):
    announce("residual norm autograd, main grads, streams, graphs")
    sets = [_operands(cuda, 24, 520, torch.bfloat16, False, True, s) for s in range(3)]

    def step(o):
        leaf = _leaves(o)
        h, y = _apply(leaf)
        keys = [k for k in ("x", "residual", "pg", "pb", "gate", "gamma", "beta")]
        return h.detach(), y.detach(), *torch.autograd.grad((h, y), [leaf[k] for k in keys], (o["dh"], o["dy"]))

    want = [step(o) for o in sets]
    o = sets[0]
    h, y, stats = _forward(o, 0.7, 1e-5, False)
    grads = _grads(o)
    dx, dres = _backward(o, stats, o["dh"], o["dy"], 0.7, 1e-5, False, grads)
    for a, b in zip(want[0], (h, y, dx, dres, *(g[0] for g in grads))):
        assert torch.equal(a, b)
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, b) for a, b in zip(step(o), want[0]))
    # any leading shape, strides and offsets; one output unused; inputs without gradients
    leaf = _leaves(o)
    for k in ("x", "residual"):
        leaf[k] = torch.empty(24 * 520 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(4, 6, 520).copy_(
            o[k].view(4, 6, 520)).transpose(0, 1).requires_grad_(True)
    hh, yy = _apply(leaf)
    assert torch.equal(hh.transpose(0, 1).reshape(24, 520), h) and torch.equal(yy.transpose(0, 1).reshape(24, 520), y)
    (got,) = torch.autograd.grad(yy, leaf["x"], o["dy"].view(4, 6, 520).transpose(0, 1))
    alone, _ = _backward(o, stats, None, o["dy"], 0.7, 1e-5, False, [None] * 5)
    assert torch.equal(got.transpose(0, 1).reshape(24, 520), alone)
    # main grads: added or, where stale, stored; one parameter in both places
    wide = _grads(o, fp32=True)
    _backward(o, stats, o["dh"], o["dy"], 0.7, 1e-5, False, wide)
    params = {k: torch.nn.Parameter(o[k].clone()) for k in ("pg", "pb", "gate", "gamma", "beta")}
    for p in params.values():
        p.main_grad = torch.ones(520, device=cuda)
    params["beta"]._eth_main_grad_stale = True
    hh, yy = _apply({**o, **params})
    torch.autograd.backward((hh, yy), (o["dh"], o["dy"]))
    for k, (g, _) in zip(("pg", "pb", "gate", "gamma", "beta"), wide):
        assert params[k].grad is None and torch.equal(params[k].main_grad, g if k == "beta" else g + 1.0)
    both = torch.nn.Parameter(o["gamma"].clone())
    both.main_grad = torch.ones(520, device=cuda)
    same = {**o, "pg": o["gamma"]}
    st2 = _forward(same, 0.7, 1e-5, False)[2]
    wide = _grads(same, fp32=True)
    _backward(same, st2, o["dh"], o["dy"], 0.7, 1e-5, False, wide)
    torch.autograd.backward(_apply({**o, "pg": both, "gamma": both}), (o["dh"], o["dy"]))
    assert torch.equal(both.main_grad, 1.0 + wide[0][0] + wide[3][0])
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(step(s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    held = {k: v.clone() for k, v in sets[0].items()}

    def captured():
        h, y, stats = _forward(held, 0.7, 1e-5, False)
        grads = _grads(held)
        dx, dres = _backward(held, stats, held["dh"], held["dy"], 0.7, 1e-5, False, grads)
        return h, y, dx, dres, *(g[0] for g in grads)

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
        for k in held:
            held[k].copy_(sets[s][k])
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want[s]))
        step(sets[(s + 1) % 3])
    empty = _operands(cuda, 0, 520, torch.bfloat16, False, True)
    leaf = _leaves(empty)
    hh, yy = _apply(leaf)
    assert hh.shape == yy.shape == (0, 520)
    assert all((g == 0).all() for g in torch.autograd.grad((hh.sum() + yy.sum()), [leaf["x"], leaf["gate"], leaf["beta"]]))


def test_refusals(cuda):
    announce("residual norm refusals")
    o = _operands(cuda, 4, 64, torch.bfloat16, False, True)
    good = dict(x=o["x"], residual=o["residual"], post_gamma=o["pg"], post_beta=o["pb"], gate=o["gate"],
                residual_scale=1.0, gamma=o["gamma"], beta=o["beta"], eps=1e-5, rms=False)
    shifted = torch.zeros(65, dtype=torch.bfloat16, device=cuda)[1:]
    for change in (dict(x=o["x"].float()), dict(residual=o["residual"].half()), dict(residual=o["residual"][:3]),
                   dict(x=o["x"][:, :60].contiguous()), dict(x=o["x"].t()), dict(post_gamma=None), dict(gamma=None),
                   dict(beta=None), dict(post_beta=None), dict(rms=True), dict(gate=o["gate"][:56]), dict(gate=shifted),
                   dict(gamma=o["gamma"].float()), dict(gate=o["gate"].cpu()), dict(residual=o["residual"].cpu()),
                   dict(residual_scale=float("nan")), dict(residual_scale=float("inf")), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(x=torch.zeros(2, 8200, dtype=torch.bfloat16, device=cuda)),
                   dict(x=o["x"].cpu(), residual=o["residual"].cpu())):
        with pytest.raises(ValueError):
            K.residual_norm_fwd(**(good | change))
    stats = K.residual_norm_fwd(**good)[2]
    for kw in (dict(dh=None, dy=None), dict(dh=o["dh"].float()), dict(dy=o["dy"][:3]), dict(stats=stats[:3]),
               dict(stats=stats.double()), dict(residual=o["residual"].half()), dict(grads=[(o["pg"].clone(), True), *[None] * 4]),
               dict(grads=[(torch.zeros(60, device=cuda), False), *[None] * 4]),
               dict(grads=[(s := torch.zeros(64, device=cuda), False), (s, False), *[None] * 3])):
        args = dict(residual=o["residual"], stats=stats, dh=o["dh"], dy=o["dy"], grads=[None] * 5) | kw
        with pytest.raises(ValueError):
            _backward({**o, "residual": args["residual"]}, args["stats"], args["dh"], args["dy"], 1.0, 1e-5, False, args["grads"])
    with pytest.raises(ValueError):
        GatedResidualNormFn.apply(o["x"], o["residual"][:2], o["pg"], o["pb"], None, 1.0, o["gamma"], o["beta"])
