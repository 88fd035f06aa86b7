"""CPU: the tile lists of packed sequences, their refusals and those of the
packed attention entry points, and the oracle against differences."""

import random

import numpy as np
import pytest
import torch

from eth_amd import _native as nat
from eth_amd import kernels as K
from eth_amd import packed as pk
from oracle.packed import packed_attention


@pytest.mark.parametrize("queries", [True, False])
@pytest.mark.parametrize("rows", [32, 64, 128])
def test_tile_lists_cover_every_row_once(rows, queries):
    rng = random.Random(rows + queries)
    for _ in range(60):
        lengths = [rng.choice((0, 1, rng.randrange(1, 700))) for _ in range(rng.randrange(0, 9))]
        total = max(1, sum(lengths) + rng.choice((0, 0, 1, 40, 300)))
        tiles, blocks = pk._tile_list(lengths, total, rows, queries)
        seen = np.zeros(total, dtype=int)
        begins = np.cumsum([0, *lengths])
        chains = []
        for t in tiles:
            begin, length, start = int(t["begin"]), int(t["len"]), int(t["start"])
            if length < 0:
                assert -length <= rows and begin >= sum(lengths) and start == 0
                seen[begin : begin - length] += 1
                continue
            i = [j for j, x in enumerate(lengths) if x and begins[j] == begin]
            assert len(i) == 1 and lengths[i[0]] == length and start % rows == 0 and start < length
            seen[begin + start : begin + min(start + rows, length)] += 1
            chains.append(-(-(min(start + rows, length) if queries else length - start) // 64))
        assert (seen == 1).all()
        assert chains == sorted(chains, reverse=True) == blocks.tolist()


def test_split_chains():
    """Split tiles are the longest, every chain fits its pieces, and no list
    whose steps fill the slots evenly is split."""
    assert pk.split_chains(np.array([], dtype=np.int64), 4, 512) == (0, 0, 0)
    assert pk.split_chains(np.full(512, 40), 1, 512) == (0, 0, 0)
    assert pk.split_chains(np.array([19]), 1, 512) == (0, 0, 0)
    assert pk.split_chains(np.array([20, 8, 3]), 1, 512) == (1, 3, 8)
    rng = random.Random(3)
    for _ in range(300):
        chain = np.array(sorted((rng.randrange(1, 300) for _ in range(rng.randrange(1, 80))), reverse=True))
        heads, slots = rng.choice((1, 2, 8, 32)), rng.choice((256, 512))
        tiles, pieces, steps = pk.split_chains(chain, heads, slots)
        if tiles:
            assert (chain[:tiles] > steps).all() and (chain[tiles:] <= steps).all()
            share = -(-chain.sum() * heads // slots)
            assert pieces > 1 and pieces * steps >= chain[0]
            assert chain[0] >= max(steps, share) + pk.WORTH_SPLITTING
            assert pk.MIN_PIECE <= steps <= max(share * 1.5, pk.MIN_PIECE)
            assert steps >= min(share, pk.GOOD_PIECE)
        else:
            share = -(-chain.sum() * heads // slots)
            assert chain[0] < max(pk.MIN_PIECE, share, min(share * 1.5, pk.GOOD_PIECE)) + pk.WORTH_SPLITTING


@pytest.mark.parametrize("lengths,total", [
    ([3, -1], None), ([3, 2.0], None), ([True], None), ([3, 4], 6), ([], None), ([0, 0], None), ([], 0),
    ([2**31], None), ([1], 2**31), (torch.ones(2, 2, dtype=torch.int64), None), (torch.ones(2), None),
])
def test_packed_sequences_refuse(lengths, total):
    with pytest.raises(ValueError):
        pk.PackedSequences(lengths, total=total)


def test_packed_sequences_need_the_gpu():
    with pytest.raises(ValueError, match="GPU"):
        pk.PackedSequences([3, 4], device="cpu")


def test_tile_rows_by_shared_heads():
    rows = lambda n, m: nat.value("eth_packed_attn_tile_rows", n, m)  # noqa: E731
    assert [rows(8, 8), rows(8, 4), rows(6, 2), rows(8, 2), rows(8, 1), rows(12, 2)] == [128, 64, 128, 32, 32, 64]
    assert [rows(8, 3), rows(0, 1), rows(4, 0), rows(2, 4)] == [0, 0, 0, 0]
    assert {rows(n, m) for m in range(1, 9) for n in range(m, 65, m)} == set(pk.QUERY_TILE_ROWS)


def _desc(**changes):
    d = nat.PackedAttnDesc()
    d.rows, d.heads, d.kv_heads, d.head_dim, d.dtype, d.scale = 16, 4, 2, 64, nat.ETH_BF16, 0.125
    for name in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        getattr(d, f"{name}_strides")[:] = (256, 64)
    d.q_tiles = d.k_tiles = 4096
    d.n_q_tiles = d.n_k_tiles = 1
    for name, value in changes.items():
        if name.endswith(("strides", "split")):
            getattr(d, name)[:] = value
        else:
            setattr(d, name, value)
    return d


@pytest.mark.parametrize("changes,match", [
    (dict(dtype=nat.ETH_F32), "bf16/fp16"), (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"), (dict(rows=0), "rows"),
    (dict(rows=2**31), "rows"), (dict(n_q_tiles=0), "tiles"), (dict(k_tiles=None), "tiles"),
    (dict(n_q_tiles=2**30), "too many"), (dict(q_split=(2, 2, 8)), "split"), (dict(k_split=(1, 1, 8)), "split"),
    (dict(q_split=(1, 2, 0)), "split"), (dict(k_split=(-1, 2, 8)), "split"), (dict(k_split=(1, 2**24, 8)), "split"), (dict(q_strides=(252, 64)), "aligned"), (dict(v_strides=(-256, 64)), "strides"),
    (dict(k_strides=(2**24, 64)), "strides"), (dict(o_strides=(256, 4)), "aligned"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
])
def test_c_entry_refuses_before_any_launch(changes, match):
    import ctypes

    d = _desc(**changes)
    p = 1 << 20
    with pytest.raises(ValueError, match=match):
        nat.call("eth_packed_attn_fwd", ctypes.byref(d), p, p, p, p, p, None, None)
    assert nat.value("eth_packed_attn_workspace", ctypes.byref(d), 0) == 0
    with pytest.raises(ValueError, match=match):
        nat.call("eth_packed_attn_bwd", ctypes.byref(d), p, p, p, p, p, p, p, p, p, p, p, None)


def test_c_entry_refuses_null_and_misaligned_pointers():
    import ctypes

    d, p = _desc(), 1 << 20
    for bad in (None, p + 8):
        for i in range(4):
            args = [p] * 5
            args[i] = bad
            with pytest.raises(ValueError):
                nat.call("eth_packed_attn_fwd", ctypes.byref(d), *args, None, None)
    with pytest.raises(ValueError, match="null"):
        nat.call("eth_packed_attn_fwd", None, p, p, p, p, p, None, None)
    d = _desc(q_split=(1, 3, 8), n_q_tiles=2)
    for ws in (None, p + 8):
        with pytest.raises(ValueError, match="workspace"):
            nat.call("eth_packed_attn_fwd", ctypes.byref(d), p, p, p, p, p, ws, None)
        with pytest.raises(ValueError, match="workspace"):
            nat.call("eth_packed_attn_bwd", ctypes.byref(d), p, p, p, p, p, p, p, p, p, p, ws, None)
    # 2 groups of heads x 3 pieces of 4 waves' 32 x 64 accumulators, 64 lanes' statistics
    assert nat.value("eth_packed_attn_workspace", ctypes.byref(d), 0) == 2 * 3 * 4 * (32 * 64 * 4 + 64 * 8)
    assert nat.value("eth_packed_attn_workspace", ctypes.byref(d), 1) == 2 * 3 * 4 * 32 * 64 * 4
    d = _desc(k_split=(1, 3, 8), head_dim=128)
    assert nat.value("eth_packed_attn_workspace", ctypes.byref(d), 0) == 0
    assert nat.value("eth_packed_attn_workspace", ctypes.byref(d), 1) == 2 * 3 * 8 * 32 * 128 * 4


def test_oracle_gradients_equal_differences():
    """Directional derivatives of sum(out * dout) in 64 bits, central
    differences with steps of 1e-5: their error is of the order of 1e-10."""
    gen = torch.Generator().manual_seed(2)
    lengths, rows, n, m, hn = [5, 0, 1, 9], 17, 6, 2, 8
    q, dout = (torch.randn(rows, n, hn, generator=gen, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(rows, m, hn, generator=gen, dtype=torch.float64) for _ in range(2))
    r = packed_attention(q, k, v, lengths, scale=0.3, dout=dout)
    assert (r["out"][15:] == 0).all() and (r["dk"][15:] == 0).all() and (r["lse"][:, 15:] == -float("inf")).all()
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn((q, k, v)[i].shape, generator=gen, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            x = [q, k, v]
            x[i] = x[i] + sign * 1e-5 * d
            ends.append((packed_attention(*x, lengths, scale=0.3)["out"] * dout).sum())
        assert abs((ends[0] - ends[1]) / 2e-5 - (r[name] * d).sum()) < 1e-7, name


def test_oracle_is_attention_of_each_sequence_alone():
    import torch.nn.functional as F

    gen = torch.Generator().manual_seed(3)
    lengths, n, m, hn = [7, 12], 4, 2, 8
    q = torch.randn(19, n, hn, generator=gen, dtype=torch.float64)
    k, v = (torch.randn(19, m, hn, generator=gen, dtype=torch.float64) for _ in range(2))
    out = packed_attention(q, k, v, lengths)["out"]
    for a, b in ((0, 7), (7, 19)):
        x = [t[a:b].transpose(0, 1).repeat_interleave(n // t.shape[1], 0) for t in (q, k, v)]
        want = F.scaled_dot_product_attention(*x, is_causal=True).transpose(0, 1)
        assert torch.allclose(out[a:b], want, atol=1e-12)


@pytest.mark.parametrize("total", [7.5, 8.0, True])
def test_total_is_a_whole_number(total):
    with pytest.raises(ValueError, match="whole"):
        pk.PackedSequences([1], total=total)


@pytest.mark.parametrize("strides,fits", [
    ((256, 64), True), ((64, 512), True), ((512, 128), True), ((64, 64), False), ((128, 64), False), ((64, 256), False),
    ((248, 64), False), ((64, 504), False), ((64, 0), False), ((0, 64), False),
])
def test_written_rows_may_not_overlap(strides, fits):
    """8 rows of 4 heads of 64: apart by rows or by heads, or refused."""
    t = torch.zeros(8192).as_strided((8, 4, 64), (*strides, 1))
    if fits:
        assert K._thd_strides("dq", t, written=True) == strides
    else:
        with pytest.raises(ValueError, match="overlap"):
            K._thd_strides("dq", t, written=True)
    assert K._thd_strides("q", t) == strides
