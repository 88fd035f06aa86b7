"""CPU: the backward passes of the logit rows take their operands as autograd
gives them back.  Hooks on saved tensors (offloading to the host and back) bring
rows that were apart back side by side: a kernel that went on from the forward's
row distance would read past their end."""

from types import SimpleNamespace

import pytest
import torch

from eth_amd import _native as nat
from eth_amd import kernels as K
from eth_amd.model.functional import TokenLogprobsFn, TopkDistillFn

ROWS, V, LD = 4, 100, 147


@pytest.fixture
def launched(monkeypatch):
    """Arguments of the launches, which do not happen."""
    calls = []
    monkeypatch.setattr(K, "_launch", lambda index, name, *args: calls.append((name, args)))
    return calls


def _saved(fn):
    """(context as after a forward of rows LD apart, its saved tensors moved
    side by side, upstream gradients)"""
    layout = -1, nat.dtype_code(torch.bfloat16), ROWS, V, LD  # (the CPU's device index)
    z, row = torch.zeros(ROWS, V, dtype=torch.bfloat16), torch.zeros(ROWS)
    ctx = SimpleNamespace(layout=layout, shape=z.shape, ignore_index=-100, temperature=1.0, teacher=torch.float32,
                          bad_flag=torch.zeros(1, dtype=torch.int32))
    if fn is TokenLogprobsFn:
        ctx.saved_tensors = z, torch.zeros(ROWS, dtype=torch.int64), torch.zeros(ROWS, 2), row
        return ctx, (row, row, None, None)
    ctx.saved_tensors = z, torch.zeros(ROWS, 3, dtype=torch.int64), torch.zeros(ROWS, 3), torch.zeros(ROWS, 4)
    return ctx, (row,)


@pytest.mark.parametrize("fn", [TokenLogprobsFn, TopkDistillFn])
def test_row_distance_is_that_of_the_saved_logits(launched, fn):
    ctx, grads = _saved(fn)
    fn.backward(ctx, *grads)
    assert launched[0][1][:2] == (ctx.saved_tensors[0].data_ptr(), V)
    apart = torch.zeros(ROWS, LD, dtype=torch.bfloat16)[:, :V]
    ctx.saved_tensors = apart, *ctx.saved_tensors[1:]
    fn.backward(ctx, *grads)
    assert launched[1][1][:2] == (apart.data_ptr(), LD)


@pytest.mark.parametrize("fn", [TokenLogprobsFn, TopkDistillFn])
def test_saved_tensors_of_another_kind_are_refused(launched, fn):
    ctx, grads = _saved(fn)
    good = ctx.saved_tensors
    z = good[0]
    swaps = [(0, z.float()), (0, z[:3]), (0, z.t().contiguous().t()), (0, z[:1].expand(ROWS, V)), (1, good[1].int()),
             (1, good[1].repeat_interleave(2, 0)[::2]), (2, good[2].double()), (3, good[3].repeat_interleave(2, 0)[::2])]
    for i, t in swaps:
        ctx.saved_tensors = *good[:i], t, *good[i + 1 :]
        with pytest.raises(ValueError):
            fn.backward(ctx, *grads)
    assert not launched


def test_packed_attention_refuses_saved_results_of_another_kind(launched):
    q = torch.zeros(8, 4, 64, dtype=torch.bfloat16)
    out, lse = torch.zeros(8, 256, dtype=torch.bfloat16), torch.zeros(4, 8)
    packed = SimpleNamespace(device=SimpleNamespace(index=-1), descriptors={})
    for o, x in ((out.half(), lse), (out.t().contiguous().t(), lse), (out, lse.double()), (out, lse.t().contiguous().t())):
        with pytest.raises(ValueError):
            K._packed_attention_grads(q, q, q, o, out, x, packed)
    assert not launched
