"""GPU: packed attention whose query chains are split where several query heads
share a workgroup, with several key and value heads and several workgroups to
each of them: the joins' rows, heads and statistics.  Bounds are those of the
other parity tests."""

import pytest
import torch

from eth_amd import _native as nat
from eth_amd.packed import QUERY_TILE_ROWS, PackedSequences
from oracle.packed import packed_attention
from tests.conftest import announce
from tests.test_gpu_packed_attention import U, _check, _inputs, _run, _split

pytestmark = pytest.mark.gpu

CASES = [
    # lengths, tail, n, m, hn: query heads that share a workgroup, and their workgroups to a key/value head
    ([2000, 5], 3, 8, 2, 64),  # 4, 1
    ([2410], 0, 16, 2, 128),  # 4, 2
    ([1500, 90], 0, 4, 2, 128),  # 2, 1
    ([1500, 0, 40], 10, 6, 1, 96),  # 2, 3
    ([753, 787, 1294], 0, 8, 4, 80),  # 2, 1
    ([1345, 1300], 0, 6, 2, 64),  # 1, 3
    ([1400], 9, 12, 2, 40),  # 2, 3
    ([3467], 0, 8, 1, 64),  # 4, 2
]


def test_cases_split_query_chains(cuda):
    """All do, and among them are 1, 2 and 4 heads a workgroup, with several
    key and value heads and several workgroups to each."""
    seen = set()
    for lengths, tail, n, m, hn in CASES:
        q_split = PackedSequences(lengths, total=sum(lengths) + tail, device=cuda).plan(n, m, hn)[4]
        assert q_split[0], (lengths, n, m)
        shared = max(QUERY_TILE_ROWS) // nat.value("eth_packed_attn_tile_rows", n, m)
        seen.add((shared, m > 1, n // shared > m))
    assert {s for s, several, _ in seen if several} == {1, 2, 4}
    assert {s for s, several, more in seen if several and more} == {1, 2, 4}


@pytest.mark.parametrize("lengths,tail,n,m,hn", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_forward_and_gradients(cuda, dtype, lengths, tail, n, m, hn):
    announce(f"packed attention split queries {dtype} {lengths} +{tail} n={n} m={m} hn={hn}")
    rows = sum(lengths) + tail
    mixed, dout = _inputs(rows, n, m, hn, dtype, rows + n + hn)
    ref = packed_attention(*(t.double() for t in _split(mixed, n, m)), lengths, dout=dout.double().view(rows, n, hn),
                           u=U[dtype])
    got = _run(*_split(mixed.to(cuda), n, m), PackedSequences(lengths, total=rows, device=cuda), dout.to(cuda))
    torch.cuda.synchronize()
    _check(got, ref, dtype)
