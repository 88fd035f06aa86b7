"""Sequences of different lengths packed into one row dimension.

`PackedSequences` is what the packed attention kernels need to know of a
batch: which rows form which sequence, as device lists of tiles (blocks of
queries, blocks of keys, and blocks of rows that no sequence covers), built and
checked once on the host and shared by every layer of the batch, forward and
backward.  The lists are ordered by the length of a tile's chain, so that the
longest start first.
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


class PackedSequences:
    """Rows [0, lengths[0]) are the first sequence, the next lengths[1] rows
    the second, and so on; rows from sum(lengths) to `total` (default: none)
    belong to no sequence.  Lengths may be zero.  Device lists are uploaded
    here (about 0.1 ms, and the host waits for the current stream), so make it
    ahead of the work that needs it and outside of a graph capture, and keep it for
    as long as a graph that was captured with it is replayed."""

    def __init__(self, lengths, total=None, device="cuda"):
        if isinstance(lengths, torch.Tensor):
            if lengths.dim() != 1 or lengths.is_floating_point() or lengths.dtype == torch.bool:
                raise ValueError("lengths must be a one-dimensional list of whole numbers")
            lengths = lengths.tolist()
        lengths = list(lengths)
        for x in lengths:
            if type(x) is not int and not isinstance(x, np.integer) or x < 0:
                raise ValueError(f"a sequence length must be a whole number of at least 0, got {x!r}")
        self.lengths = tuple(int(x) for x in lengths)
        covered = sum(self.lengths)
        if isinstance(total, (bool, float)):
            raise ValueError(f"total must be a whole number, got {total!r}")
        self.total = covered if total is None else operator.index(total)
        if not covered <= self.total or not 0 < self.total < 2**31:
            raise ValueError(f"total must be at least 1, at least the {covered} rows of the sequences, and below 2^31 "
                             f"(got {self.total})")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("packed sequences live on the GPU (no CPU fallback)")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        lists = {rows: _tile_list(self.lengths, self.total, rows, True) for rows in QUERY_TILE_ROWS}
        lists["keys"] = _tile_list(self.lengths, self.total, KEY_TILE_ROWS, False)
        self._table = nat.table_to_device(np.concatenate([tiles for tiles, _ in lists.values()]), self.device)
        self._home = nat.stream_ptr(self.device)
        self._chains = {key: chain for key, (_, chain) in lists.items()}
        self._at, at = {}, self._table.data_ptr()
        for key, (tiles, _) in lists.items():
            self._at[key] = (at, tiles.size)
            at += tiles.nbytes
        self._plans = {}
        self.descriptors = {}  # of calls with this plan, by shapes and strides

    def in_use(self):
        """A launch on the current stream is about to read the lists."""
        if torch._C._cuda_getCurrentRawStream(self.device.index) != self._home:
            if not torch.cuda.is_current_stream_capturing():
                self._table.record_stream(torch.cuda.current_stream(self.device))

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
