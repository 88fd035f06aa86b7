"""Sequences and tasks of different lengths packed into one row dimension.

`PackedSequences` is what the packed attention kernels need to know of a
batch: which rows form which sequence, as device lists of tiles (blocks of
queries, blocks of keys, and blocks of rows that no sequence covers), built and
checked once on the host and shared by every layer of the batch, forward and
backward.  The lists are ordered by the length of a tile's chain, so that the
longest start first.

`AdapterRows` is the same for low-rank adapters: which rows use which adapter.
"""

import operator

import numpy as np
import torch

from . import _native as nat

KEY_TILE_ROWS = 128  # keys per workgroup of the dK/dV kernels
QUERY_TILE_ROWS = (32, 64, 128)  # queries per workgroup, by the heads that share one
BLOCK_ROWS = 64  # keys (queries) of a step of a query (key) tile
MIN_PIECE = 8  # steps of a split tile's piece, at least
GOOD_PIECE = 28  # and where the work fills the slots several times over
WORTH_SPLITTING = 12  # steps that a split has to save


def _tile_list(lengths, total, rows, queries):
    """(eth_packed_tile entries of `rows` rows, the 64-row blocks of each
    one's chain): a query tile's chain grows with its end in the sequence, a
    key tile's with what is left behind its start."""
    lengths = np.asarray(lengths, dtype=np.int64).reshape(-1)
    begins = np.cumsum(lengths) - lengths
    counts = -(-lengths // rows)
    seq = np.repeat(np.arange(lengths.size), counts)
    start = (np.arange(seq.size) - np.repeat(np.cumsum(counts) - counts, counts)) * rows
    chain = -(-(np.minimum(start + rows, lengths[seq]) if queries else lengths[seq] - start) // BLOCK_ROWS)
    order = np.argsort(-chain, kind="stable")
    covered = int(lengths.sum())
    spare = np.arange(covered, total, rows)  # rows behind the last sequence
    tiles = np.zeros(seq.size + spare.size, dtype=nat.PACKED_TILE_DTYPE)
    tiles["begin"] = np.concatenate([begins[seq][order], spare])
    tiles["len"] = np.concatenate([lengths[seq][order], -np.minimum(rows, total - spare)])
    tiles["start"][: seq.size] = start[order]
    return tiles, chain[order]


def split_chains(chain, heads, slots):
    """(tiles, pieces, steps) of a list whose `chain` steps (longest first) are
    run for `heads` heads each on `slots` workgroups at a time: (0, 0, 0) where
    no tile is worth splitting.

    The list ends no earlier than its longest chain, nor than its steps spread
    over the slots.  Where the first is well above the second, chains are cut:
    into pieces of half as much again as the second, whose partial sums cost less
    than its own would, or where that is long into smaller ones, which fill the
    slots more evenly until their partial sums cost more.  Backward of 16384 rows,
    8 heads of 64 on one, 258 steps a slot (us): uncut 3006, pieces of 258 1198, 129
    1072, 86 1018, 65 1012, 43 1021; of 8192 packed rows, 16 heads of 128 on four, 53
    steps a slot: 295, 53 254, 27 248, 18 268; of 8192 rows of one head of 128, 9 and
    17 steps a slot, pieces of 9 and 17 145, of 13 and 25 112; of 3 x 1311 rows, 32
    heads of 80 on eight, 23 steps, pieces of 23 195, of 28 170."""
    if not chain.size:
        return 0, 0, 0
    share = -(-int(chain.sum()) * heads // slots)
    steps = max(MIN_PIECE, min(share * 3 // 2, max(GOOD_PIECE, share * 2 // 7)))
    longest = int(chain[0])
    if longest < max(share, steps) + WORTH_SPLITTING:
        return 0, 0, 0
    return int(np.searchsorted(-chain, -steps, side="left")), -(-longest // steps), steps


def _checked_lengths(lengths, what):
    if isinstance(lengths, torch.Tensor):
        if lengths.dim() != 1 or lengths.is_floating_point() or lengths.dtype == torch.bool:
            raise ValueError("lengths must be a one-dimensional list of whole numbers")
        lengths = lengths.tolist()
    lengths = list(lengths)
    for x in lengths:
        if type(x) is not int and not isinstance(x, np.integer) or x < 0:
            raise ValueError(f"a {what} length must be a whole number of at least 0, got {x!r}")
    return tuple(int(x) for x in lengths)


def _checked_total(total, covered, what):
    if isinstance(total, (bool, float)):
        raise ValueError(f"total must be a whole number, got {total!r}")
    total = covered if total is None else operator.index(total)
    if not covered <= total or not 0 < total < 2**31:
        raise ValueError(f"total must be at least 1, at least the {covered} rows of the {what}, and below 2^31 "
                         f"(got {total})")
    return total


def _checked_device(device, what):
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"{what} live on the GPU (no CPU fallback)")
    return device if device.index is not None else torch.device("cuda", torch.cuda.current_device())


class _DeviceLists:
    """Lists of a batch's rows in device memory, uploaded once."""

    def _upload(self, table):
        self._table = nat.table_to_device(table, self.device)
        self._home = nat.stream_ptr(self.device)

    def in_use(self):
        """A launch on the current stream is about to read the lists."""
        if torch._C._cuda_getCurrentRawStream(self.device.index) != self._home:
            if not torch.cuda.is_current_stream_capturing():
                self._table.record_stream(torch.cuda.current_stream(self.device))


class PackedSequences(_DeviceLists):
    """Rows [0, lengths[0]) are the first sequence, the next lengths[1] rows
    the second, and so on; rows from sum(lengths) to `total` (default: none)
    belong to no sequence.  Lengths may be zero.  Device lists are uploaded
    here (about 0.1 ms, and the host waits for the current stream), so make it
    ahead of the work that needs it and outside of a graph capture, and keep it for
    as long as a graph that was captured with it is replayed."""

    def __init__(self, lengths, total=None, device="cuda"):
        self.lengths = _checked_lengths(lengths, "sequence")
        self.total = _checked_total(total, sum(self.lengths), "sequences")
        self.device = _checked_device(device, "packed sequences")
        lists = {rows: _tile_list(self.lengths, self.total, rows, True) for rows in QUERY_TILE_ROWS}
        lists["keys"] = _tile_list(self.lengths, self.total, KEY_TILE_ROWS, False)
        self._upload(np.concatenate([tiles for tiles, _ in lists.values()]))
        self._chains = {key: chain for key, (_, chain) in lists.items()}
        self._at, at = {}, self._table.data_ptr()
        for key, (tiles, _) in lists.items():
            self._at[key] = (at, tiles.size)
            at += tiles.nbytes
        self._plans = {}
        self.descriptors = {}  # of calls with this plan, by shapes and strides

    def plan(self, heads, kv_heads, head_dim):
        """(query list address and count, key list address and count, query
        split, key split) for these heads."""
        plan = self._plans.get((heads, kv_heads, head_dim))
        if plan is None:
            rows = nat.value("eth_packed_attn_tile_rows", heads, kv_heads)
            cus = torch.cuda.get_device_properties(self.device).multi_processor_count
            # query workgroups a compute unit: two (where a third fits, at a head dim of 64, it
            # shares the same pipes: filling its slots too by splitting took 333 us, not 308, of
            # 16384 rows of 8 heads on one); of dK/dV two up to a head dim of 96, one above
            q_split = split_chains(self._chains[rows], heads * rows // 128, 2 * cus)
            k_split = split_chains(self._chains["keys"] * (heads // kv_heads), kv_heads, (1 if head_dim > 96 else 2) * cus)
            plan = self._plans[heads, kv_heads, head_dim] = (*self._at[rows], *self._at["keys"], q_split, k_split)
        return plan


# Tiles of a partial gradient sum, and how many sums a batch is cut into. Short
# sums fill the GPU and are long to join: [16384, 4096 -> 4096] of rank 128 takes
# 177 us of gradients so, 205 with at most 32 tiles, 272 with 16; [3000, 4096 ->
# 4096] of rank 64 37 us, 40 with 32 tiles at least, 52 with 4.
MIN_CHUNK, MAX_CHUNK, CHUNKS = 16, 128, 8


def adapter_tiles(lengths, ids, scales, rows=nat.ADAPTER_TILE_ROWS):
    """(tiles, chunks, first_chunk, used) of segments of the given lengths, adapter
    ids (-1: none) and scales: up to `rows` rows of one segment a tile, ordered by
    adapter; runs of tiles of one adapter, whose gradients are summed together;
    where each adapter's chunks start; and the adapters that have rows."""
    lengths, ids = np.asarray(lengths, dtype=np.int64).reshape(-1), np.asarray(ids, dtype=np.int64).reshape(-1)
    begins = np.cumsum(lengths) - lengths
    counts = np.where(ids >= 0, -(-lengths // rows), 0)
    seg = np.repeat(np.arange(lengths.size), counts)
    start = (np.arange(seg.size) - np.repeat(np.cumsum(counts) - counts, counts)) * rows
    order = np.argsort(ids[seg], kind="stable")
    seg, start = seg[order], start[order]
    tiles = np.zeros(seg.size, dtype=nat.ADAPTER_TILE_DTYPE)
    tiles["row"], tiles["rows"] = begins[seg] + start, np.minimum(rows, lengths[seg] - start)
    tiles["adapter"], tiles["scale"] = ids[seg], np.asarray(scales, dtype=np.float32).reshape(-1)[seg]
    per = max(MIN_CHUNK, min(MAX_CHUNK, -(-seg.size // CHUNKS)))
    used, first, many = np.unique(tiles["adapter"], return_index=True, return_counts=True)
    pieces = -(-many // per)
    chunks = np.zeros(int(pieces.sum()), dtype=nat.ADAPTER_CHUNK_DTYPE)
    at = (np.arange(chunks.size) - np.repeat(np.cumsum(pieces) - pieces, pieces)) * per
    chunks["first"] = np.repeat(first, pieces) + at
    chunks["tiles"] = np.minimum(per, np.repeat(many, pieces) - at)
    listed = int(used[-1]) + 1 if used.size else 0
    first_chunk = np.zeros(listed + 1, dtype=np.int32)
    first_chunk[used.astype(np.int64) + 1] = pieces
    return tiles, chunks, np.cumsum(first_chunk, dtype=np.int32), used.astype(np.int32)


class AdapterRows(_DeviceLists):
    """Rows [0, lengths[0]) use adapter ids[0] with scales[0] (default: one), the
    next lengths[1] rows ids[1], and so on; id -1, and rows from sum(lengths) to
    `total` (default: none), use no adapter.  Lengths may be zero, and an adapter
    may serve several segments.  Device lists are uploaded here (the host waits for
    the current stream), so make it ahead of the work that needs it and outside of a
    graph capture, and keep it for as long as a graph that was captured with it is
    replayed."""

    def __init__(self, lengths, ids, scales=None, total=None, device="cuda"):
        self.lengths = _checked_lengths(lengths, "segment")
        ids = ids.tolist() if isinstance(ids, torch.Tensor) else list(ids)
        scales = [1.0] * len(ids) if scales is None else scales.tolist() if isinstance(scales, torch.Tensor) else list(scales)
        if not len(ids) == len(scales) == len(self.lengths):
            raise ValueError(f"{len(self.lengths)} segments, {len(ids)} ids and {len(scales)} scales do not match")
        for x in ids:
            if type(x) is not int and not isinstance(x, np.integer) or not -1 <= x < 65535:
                raise ValueError(f"an adapter id must be -1 or a whole number from 0 to 65534, got {x!r}")
        self.ids, self.scales = tuple(int(x) for x in ids), tuple(float(x) for x in scales)
        if not all(abs(x) <= 2.0**64 for x in self.scales):
            raise ValueError("scales must be finite, up to 2^64")
        self.total = _checked_total(total, sum(self.lengths), "segments")
        self.device = _checked_device(device, "adapter rows")
        tiles, chunks, first_chunk, used = adapter_tiles(self.lengths, self.ids, self.scales)
        of_row = np.full(self.total, -1, dtype=np.int32)
        of_row[: sum(self.lengths)] = np.repeat(np.asarray(self.ids, dtype=np.int32), self.lengths)
        self.n_tiles, self.n_chunks, self.n_used, self.n_listed = tiles.size, chunks.size, used.size, first_chunk.size - 1
        if self.n_tiles >= 2**23 or self.n_chunks >= 2**16:
            raise ValueError(f"{self.n_tiles} tiles in {self.n_chunks} sums are too many for one call")
        parts = [tiles, chunks, first_chunk, used, of_row]
        self._upload(np.concatenate([np.ascontiguousarray(x).view(np.uint8) for x in parts]))
        at = self._table.data_ptr()
        self.addresses = []  # of tiles, chunks, first_chunk, used and of_row
        for x in parts:
            self.addresses.append(at)
            at += x.nbytes
