"""CPU: packed attention refuses lists whose workgroups have 2^32 threads and
more in all, which a launch would take modulo 2^32 without an error."""

import ctypes

import pytest

from eth_amd import _native as nat

P = 1 << 20


def _desc(heads, kv_heads, head_dim, q_tiles, k_tiles, **splits):
    d = nat.PackedAttnDesc()
    d.rows, d.heads, d.kv_heads, d.head_dim, d.dtype, d.scale = 2**25, heads, kv_heads, head_dim, nat.ETH_BF16, 0.125
    for name in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        getattr(d, f"{name}_strides")[:] = (heads * 128, 128)
    d.q_tiles = d.k_tiles = 4096
    d.n_q_tiles, d.n_k_tiles = q_tiles, k_tiles
    for name, value in splits.items():
        getattr(d, name)[:] = value
    return ctypes.byref(d)


@pytest.mark.parametrize("args,splits", [
    ((1, 1, 64, 2**24, 1), {}),  # 2^24 workgroups of 256
    ((8, 8, 64, 2**21, 1), {}),
    ((16, 4, 64, 2**22, 1), {}),  # four heads a workgroup
    ((1, 1, 64, 1, 2**24), {}),
    ((4, 2, 128, 1, 2**22), {}),  # of 512
    ((1, 1, 64, 2**24 - 2, 1), dict(q_split=(1, 3, 8))),  # with the pieces of split tiles
])
def test_too_many_workgroups_are_refused(args, splits):
    d = _desc(*args, **splits)
    with pytest.raises(ValueError, match="too many tiles"):
        nat.call("eth_packed_attn_fwd", d, P, P, P, P, P, P, None)
    with pytest.raises(ValueError, match="too many tiles"):
        nat.call("eth_packed_attn_bwd", d, *[P] * 11, None)
    assert nat.value("eth_packed_attn_workspace", d, 1) == 0


def test_the_most_that_a_launch_takes_is_not_refused():
    """(seen by the next refusal: no launch)"""
    for args in ((1, 1, 64, 2**24 - 1, 2**24 - 1), (16, 4, 128, 2**22 - 1, 2**21 - 1)):
        with pytest.raises(ValueError, match="null"):
            nat.call("eth_packed_attn_fwd", _desc(*args), None, P, P, P, P, P, None)
