"""CPU: the lists of rows and their adapters, their refusals and those of the
adapter entry points before any launch, and the oracle against differences."""

import ctypes
import random

import numpy as np
import pytest
import torch

from eth_amd import _native as nat
from eth_amd import packed as pk
from oracle.adapters import adapter_linear

P = 1 << 20


def test_lists_cover_every_adapted_row_once():
    rng = random.Random(5)
    for _ in range(200):
        lengths = [rng.choice((0, 1, rng.randrange(1, 900))) for _ in range(rng.randrange(0, 12))]
        ids = [rng.randrange(-1, rng.choice((1, 3, 20))) for _ in lengths]
        scales = [rng.uniform(-2, 2) for _ in lengths]
        tiles, chunks, first_chunk, used = pk.adapter_tiles(lengths, ids, scales)
        of_row = np.repeat(np.array([*ids, -1]), [*lengths, 0])
        scale = np.repeat(np.array([*scales, 0.0], dtype=np.float32), [*lengths, 0])
        seen = np.full(of_row.size, -1)
        for t in tiles:
            at = slice(int(t["row"]), int(t["row"] + t["rows"]))
            assert 0 < t["rows"] <= nat.ADAPTER_TILE_ROWS and (seen[at] == -1).all()
            seen[at] = t["adapter"]
            assert (scale[at] == t["scale"]).all()
        assert (seen == of_row).all()
        assert (np.diff(tiles["adapter"]) >= 0).all()
        # chunks: all tiles in order, each of one adapter
        assert np.concatenate([np.arange(c["first"], c["first"] + c["tiles"]) for c in chunks] or [[]]).tolist() == list(
            range(tiles.size))
        assert used.tolist() == sorted(set(of_row.tolist()) - {-1}) and first_chunk[0] == 0
        assert first_chunk.size == (used[-1] + 2 if used.size else 1) and first_chunk[-1] == chunks.size
        for a in range(first_chunk.size - 1):
            for c in chunks[first_chunk[a] : first_chunk[a + 1]]:
                assert 0 < c["tiles"] <= pk.MAX_CHUNK
                assert (tiles["adapter"][c["first"] : c["first"] + c["tiles"]] == a).all()


@pytest.mark.parametrize("args", [
    dict(lengths=[3, -1], ids=[0, 0]), dict(lengths=[3.0], ids=[0]), dict(lengths=[True], ids=[0]),
    dict(lengths=[3], ids=[0, 1]), dict(lengths=[3], ids=[-2]), dict(lengths=[3], ids=[65535]), dict(lengths=[3], ids=[0.0]),
    dict(lengths=[3], ids=[0], scales=[1.0, 2.0]), dict(lengths=[3], ids=[0], scales=[float("nan")]),
    dict(lengths=[3], ids=[0], scales=[float("inf")]), dict(lengths=[3], ids=[0], scales=[2.0**65]),
    dict(lengths=[3], ids=[0], total=2), dict(lengths=[0], ids=[0]), dict(lengths=[3], ids=[0], total=3.0),
    dict(lengths=[3], ids=[0], total=2**31), dict(lengths=[3], ids=[0], device="cpu"),
    dict(lengths=torch.tensor([1.0]), ids=[0]), dict(lengths=[], ids=[]),
])
def test_rows_refuse(args):
    with pytest.raises((ValueError, TypeError)):
        pk.AdapterRows(**args)


def _desc(**change):
    d = nat.AdapterDesc()
    good = dict(rows=64, in_=128, out=256, ldx=128, ldw=128, tiles=P, chunks=P, first_chunk=P, used=P, of_row=P, n_tiles=2,
                n_chunks=1, n_used=1, n_listed=1, adapters=2, rank=16, dtype=nat.ETH_BF16)
    for k, v in (good | change).items():
        setattr(d, k, v)
    return d


def test_c_entries_refuse_before_any_launch():
    def fwd(desc, **change):
        args = dict(x=P, w=P, bias=P, a=P, b=P, y=P, ut=P, scale=P, ws=P, stream=None) | change
        nat.call("eth_adapter_linear_fwd", ctypes.byref(desc) if desc else None, *args.values())

    def bwd(desc, da=(P, 0, 0), db=(2 * P, 0, 0), **change):
        grads = [ctypes.byref(nat.AdapterGrad(*g)) if g else None for g in (da, db)]
        args = dict(x=P, w=P, a=P, b=P, dy=P, ut=P, scale=P, dx=P, da=grads[0], db=grads[1], ws=P, stream=None) | change
        nat.call("eth_adapter_linear_bwd", ctypes.byref(desc) if desc else None, *args.values())

    for call in (fwd, bwd):
        with pytest.raises(ValueError):
            call(None)
        for change in (dict(dtype=nat.ETH_F32), dict(rows=0), dict(in_=0), dict(in_=124), dict(out=0), dict(out=250),
                       dict(rank=0), dict(rank=12), dict(rank=136), dict(ldx=120), dict(ldw=132), dict(adapters=0),
                       dict(n_used=2), dict(n_listed=3), dict(n_tiles=-1), dict(n_chunks=0), dict(n_tiles=0),
                       dict(n_chunks=65536), dict(tiles=None), dict(chunks=None), dict(of_row=None), dict(used=None),
                       dict(first_chunk=None), dict(rows=2**24), dict(ldx=2**26), dict(ldw=2**24), dict(n_tiles=2**23)):
            with pytest.raises(ValueError):
                call(_desc(**change))
            assert nat.value("eth_adapter_linear_workspace", ctypes.byref(_desc(**change)), 0) == -1
    for change in (dict(x=None), dict(w=None), dict(a=None), dict(b=None), dict(y=None), dict(ws=None), dict(x=P + 2),
                   dict(y=P + 8), dict(ws=P + 16), dict(ut=P + 4)):
        with pytest.raises(ValueError):
            fwd(_desc(), **change)
    with pytest.raises(ValueError):
        fwd(_desc(dtype=nat.ETH_F16), scale=None)
    for change in (dict(dy=None), dict(dx=None, da=(0, 0, 0), db=(0, 0, 0)), dict(ut=None), dict(da=None), dict(db=None),
                   dict(da=(P, 0, 1)), dict(db=(P + 4, 1, 0)), dict(db=(P, 0, 0)), dict(dy=P + 2), dict(ws=P + 8)):
        with pytest.raises(ValueError):
            bwd(_desc(), **change)


def test_structures():
    assert ctypes.sizeof(nat.AdapterDesc) == 112 and ctypes.sizeof(nat.AdapterGrad) == 16
    assert nat.ADAPTER_TILE_DTYPE.itemsize == 16 and nat.ADAPTER_CHUNK_DTYPE.itemsize == 8
    ws = lambda b, **c: nat.value("eth_adapter_linear_workspace", ctypes.byref(_desc(**c)), b)  # noqa: E731
    assert ws(0) == 64 * 32 * 2 + 256 and ws(1, n_tiles=0, n_chunks=0, n_used=0) > 0


def _slope(f, x, d):
    return (f(x + 1e-5 * d) - f(x - 1e-5 * d)) / 2e-5


def test_oracle_gradients_equal_differences():
    """Central differences in 64 bits with steps of 1e-5: off by about 1e-9."""
    gen = torch.Generator().manual_seed(4)
    randn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    v = dict(x=randn(7, 6), w=randn(5, 6), bias=randn(5), lora_a=randn(3, 4, 6), lora_b=randn(3, 5, 4))
    of_row, scale = torch.tensor([1, 1, -1, 0, 1, 0, -1]), torch.tensor([2.0, 2.0, 1.0, 0.5, 1.0, 0.5, 1.0])
    dy = randn(7, 5)
    r = adapter_linear(**v, of_row=of_row, scale=scale, dy=dy)
    for key, name in (("x", "dx"), ("lora_a", "da"), ("lora_b", "db")):
        d = randn(*v[key].shape)
        slope = _slope(lambda t: (adapter_linear(**{**v, key: t}, of_row=of_row, scale=scale)["y"] * dy).sum(), v[key], d)
        assert abs(slope - (r[name] * d).sum()) < 1e-7
    assert (r["da"][2] == 0).all() and torch.allclose(r["y"][2], v["x"][2] @ v["w"].T + v["bias"])
