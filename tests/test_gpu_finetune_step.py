"""GPU: adapters, residual norms and the loss without logits run together, as a
fine-tuning step on packed rows of several tasks: every operator's gradient is the
next one's upstream gradient.  Checked against the oracles in 64 bits on each
operator's own operands, by hand, and captured and replayed."""

import pytest
import torch

from eth_amd import kernels as K
from eth_amd.model.functional import AdapterLinearFn, GatedResidualNormFn, LinearCrossEntropyFn
from eth_amd.packed import AdapterRows
from oracle import residual_norm
from oracle.adapters import adapter_linear
from oracle.linear_xent import linear_xent
from tests.conftest import announce

pytestmark = pytest.mark.gpu

LENS, IDS, SCALES, TAIL = [37, 1, 0, 90, 55], [1, 0, 2, -1, 1], [2.0, 1.0, 1.0, 1.0, 0.5], 9
ROWS, H, V, R, ADAPTERS = sum(LENS) + TAIL, 136, 1001, 16, 3
U, LEAST, FLOOR = ({torch.bfloat16: a, torch.float16: b} for a, b in
                   ((2.0**-8, 2.0**-11), (2.0**-126, 2.0**-25), (0.0, 2.0**-37)))
LEAVES = ("x", "a", "b", "pg", "pb", "gate", "gamma", "beta", "head")


def _inputs(cuda, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    v = dict(x=randn(ROWS, H), w=randn(H, H) / H**0.5, bias=0.1 * randn(H), a=randn(ADAPTERS, R, H) / H**0.5,
             b=0.3 * randn(ADAPTERS, H, R) / R**0.5, pg=1 + 0.2 * randn(H), pb=0.1 * randn(H), gate=0.6 + 0.2 * randn(H),
             gamma=1 + 0.2 * randn(H), beta=0.1 * randn(H), head=randn(V, H) * 2 / H**0.5)
    v = {k: t.to(dtype).to(cuda) for k, t in v.items()}
    labels = torch.randint(0, V, (ROWS,), generator=gen)
    labels[:30], labels[ROWS - TAIL :] = -100, -100  # a prompt, and rows of no task
    return v, labels.to(cuda), torch.full((ROWS,), 2.0**-7, device=cuda)


def _step(v, rows, labels, dloss, bad):
    v = {k: t.detach().requires_grad_(k in LEAVES) for k, t in v.items()}
    z = AdapterLinearFn.apply(v["x"], v["w"], v["bias"], v["a"], v["b"], rows)
    h, y = GatedResidualNormFn.apply(z, v["x"], v["pg"], v["pb"], v["gate"], 0.5, v["gamma"], v["beta"])
    loss = LinearCrossEntropyFn.apply(y, v["head"], labels, bad)
    grads = torch.autograd.grad(loss, [z, h, y, *(v[k] for k in LEAVES)], dloss, allow_unused=True)
    return [t.detach() for t in (z, h, y, loss)], grads


def _within(got, r, name):
    off, bound = (got.double() - r[name]).abs(), r["bound_" + name]
    assert not got.isnan().any() and not (off > bound).any(), f"{name}: {(off / bound).max():.2f} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_step(cuda, dtype):
    announce(f"fine-tuning step {dtype}")
    rows = AdapterRows(LENS, IDS, SCALES, ROWS, cuda)
    v, labels, dloss = _inputs(cuda, dtype)
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    (z, h, y, loss), (dz, _, dy, *grads) = _step(v, rows, labels, dloss, bad)
    got = dict(zip(LEAVES, grads))
    u, least, floor = U[dtype], LEAST[dtype], FLOOR[dtype]
    counts = torch.tensor([*LENS, TAIL], device=cuda)
    of_row = torch.tensor([*IDS, -1], device=cuda).repeat_interleave(counts)
    scale = torch.tensor([*SCALES, 1.0], device=cuda).repeat_interleave(counts)
    # each operator on the operands that the others gave it
    r = linear_xent(y, v["head"], labels, -100, dloss, u, least, floor)
    _within(loss, r, "loss")
    _within(dy, {"dy": r["dh"], "bound_dy": r["bound_dh"]}, "dy")
    _within(got["head"], {"head": r["dw"], "bound_head": r["bound_dw"]}, "head")
    r = residual_norm.forward(z, v["x"], v["pg"], v["pb"], v["gate"], 0.5, v["gamma"], v["beta"], 1e-5, False, u, least)
    _within(h, r, "h")
    _within(y, r, "y")
    r = residual_norm.backward(z, v["x"], None, dy, v["pg"], v["pb"], v["gate"], 0.5, v["gamma"], 1e-5, False, u, least)
    _within(dz, {"dz": r["dx"], "bound_dz": r["bound_dx"]}, "dz")
    for k, name in (("pg", "dpost_gamma"), ("pb", "dpost_beta"), ("gate", "dgate"), ("gamma", "dgamma"), ("beta", "dbeta")):
        _within(got[k], r, name)
    dres = r["dresidual"], r["bound_dresidual"]
    r = adapter_linear(v["x"], v["w"], v["bias"], v["a"], v["b"], of_row, scale, dz, u, least, floor)
    _within(z, r, "y")
    _within(got["a"], r, "da")
    _within(got["b"], r, "db")
    # x is the block's input and its residual: autograd adds two 16-bit gradients
    total = r["dx"] + dres[0]
    _within(got["x"], {"x": total, "bound_x": r["bound_dx"] + dres[1] + 1.001 * u * total.abs() + least}, "x")
    # by hand, the same bits
    lse = K.linear_xent_fwd(y, v["head"], labels, bad)[1]
    dy2, dhead = K.linear_xent_bwd(y, v["head"], labels, lse, dloss)
    assert torch.equal(dy2, dy) and torch.equal(dhead, got["head"]) and bad.item() == 0
    _, saved = K.adapter_linear_fwd(v["x"], v["w"], v["bias"], v["a"], v["b"], rows, save=True)
    da, db = torch.empty_like(v["a"]), torch.empty_like(v["b"])
    K.adapter_linear_bwd(v["x"], v["w"], v["a"], v["b"], dz, rows, saved, False, (da, False), (db, False))
    assert torch.equal(da, got["a"]) and torch.equal(db, got["b"])
    # rows that are not scored give no gradient, adapter 2 has no rows
    quiet = labels == -100
    assert (dy[quiet] == 0).all() and (got["x"][quiet] == 0).all() and (got["a"][2] == 0).all()


def test_captured_step(cuda):
    announce("captured fine-tuning step")
    rows = AdapterRows(LENS, IDS, SCALES, ROWS, cuda)
    sets = [_inputs(cuda, torch.bfloat16, s) for s in range(3)]
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)

    def flat(v, labels, dloss):
        out, grads = _step(v, rows, labels, dloss, bad)
        return [*out, *(g for g in grads if g is not None)]

    want = [flat(*s) for s in sets]
    held = ({k: t.clone() for k, t in sets[0][0].items()}, sets[0][1].clone(), sets[0][2].clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        flat(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flat(*held)
    for s in (0, 1, 2, 1, 0):
        for k in held[0]:
            held[0][k].copy_(sets[s][0][k])
        held[1].copy_(sets[s][1])
        held[2].copy_(sets[s][2])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[s]))
        flat(*sets[(s + 1) % 3])
