"""CPU: the pieces of the vocabulary that the linear head's cross entropy takes in
its backward.  A launch reaches a piece's weights by 32-bit offsets whose upper half
stands for "not there, zero": every piece, the last and longest too, lies within 2 GiB."""

import itertools

import pytest

from eth_amd import _native as nat

REACH = 2**31 - 1


def _columns(rows, hidden, vocab, ldw):
    """At least so many columns the longest piece has, by the workspace (lists, the
    rows of h, and dz [rows, the longest piece in 8s], each in 256s)."""
    n = 2 * rows if rows <= 64 else rows
    room = lambda b: -(-b // 256) * 256  # noqa: E731
    rest = room(12) + 8 * room(4 * n) + room(2 * n * hidden)
    dz = nat.value("eth_linear_xent_workspace", rows, hidden, vocab, ldw, 2) - rest
    assert dz >= 2 * n * min(vocab, 256)
    return max(min(vocab, 256), (dz - 255) // (2 * n) - 7)


@pytest.mark.parametrize("hidden", [64, 2048, 4096, 5376, 8192, 12288, 16384, 65536])
def test_pieces_lie_within_reach(hidden):
    for rows, vocab in itertools.product((1, 33, 64, 65, 128, 500, 700, 1024, 1500, 2048, 8192, 16384),
                                         (1, 257, 32000, 50304, 65537, 100000, 128000, 131073, 152064, 196609, 262144, 2**24)):
        if rows * hidden > 2**30:
            continue
        for ldw in {hidden, hidden + 8, 2 * hidden, 32768 if hidden < 32768 else hidden}:
            columns = _columns(rows, hidden, vocab, ldw)
            assert 2 * ((columns - 1) * ldw + hidden) <= REACH, (rows, hidden, vocab, ldw, columns)


def _call(name, rows, hidden, vocab, ldw, h):
    P = 1 << 20
    last = (rows, hidden, vocab, P, nat.ETH_BF16, None) if name.endswith("fwd") else (rows, hidden, vocab, nat.ETH_BF16, None)
    first = (h, hidden, P, ldw, P, -100, P, P)
    nat.call(name, *first, *((P,) if name.endswith("fwd") else (P, P, nat.ETH_BF16, 0, P)), *last)


@pytest.mark.parametrize("name", ["eth_linear_xent_fwd", "eth_linear_xent_bwd"])
def test_weights_too_far_apart_are_refused(name):
    """256 rows of W, the least that a launch takes, within 2 GiB; what is within
    is refused for its null operand alone, ahead of any launch."""
    for vocab, ldw in ((256, 2**22 + 2**15), (300, 2**22 + 2**15), (50304, 2**23), (2**24, 2**40), (2, 2**30 - 64), (2, 2**62)):
        with pytest.raises(ValueError, match="apart"):
            _call(name, 4, 64, vocab, ldw, 1 << 20)
    for vocab, ldw in ((1, 2**40), (2, 2**30 - 72), (256, 2**22), (50304, 2**22)):
        with pytest.raises(ValueError, match="null"):
            _call(name, 4, 64, vocab, ldw, None)


def test_stated_workspace():
    """Without dh: a piece of dz, whole ones of 256 MiB (or of 256 columns, 512 bytes
    a row) and a last one half as long again, a copy of h, and the lists."""
    worst = 0.0
    for rows, vocab in itertools.product((1, 64, 65, 1000, 2047, 2048, 4096, 8192, 16384, 30000, 2**19, 2**21 - 1),
                                         (1, 1000, 24575, 24576, 50257, 98303, 151936, 262143, 2**20)):
        for hidden in (64, 512, 2048, 4096):
            n = 2 * rows if rows <= 64 else rows
            lists = 8 * (4 * n + 256) + 512
            dz = nat.value("eth_linear_xent_workspace", rows, hidden, vocab, hidden, 2) - lists - 2 * n * hidden
            most = max(384 << 20, 768 * n) + 16 * n
            assert dz <= most, (rows, hidden, vocab, dz >> 20)
            worst = max(worst, dz / most)
    assert worst > 0.9
