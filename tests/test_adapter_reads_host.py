"""CPU: the adapters' gradient kernel has a tile's x A^T and dy B in fragments of 16,
32, 64 or 128 ranks, and the tile in memory ends at the next multiple of 32: of 72 to
96 ranks, the fragments end behind it.  Every vector load of the kernel therefore
goes through a resource of its operand's size, as the assembly shows."""

import re
import subprocess

import pytest

from eth_amd import build as eb


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "adapters.s"
    subprocess.run([eb.hipcc_path(), *eb.HIPCC_FLAGS, f"-I{eb.INCLUDE}", "--cuda-device-only", "-S",
                    str(eb.CSRC / "adapters.hip"), "-o", str(out)], check=True, capture_output=True, timeout=300)
    bodies = re.findall(r"^_ZN3eth20adapter_outer_kernelILi(\d+)ELb\dE\w+:.*?\n(.*?)^\.Lfunc_end", out.read_text(), re.M | re.S)
    return [(16 * int(blocks), body) for blocks, body in bodies]


def test_fragments_end_behind_some_tiles(kernels):
    held = sorted({ranks for ranks, _ in kernels})
    past = [r for r in range(8, 129, 8) if min(h for h in held if h >= r) > -(-r // 32) * 32]
    assert len(kernels) == 2 * len(held) and past == [72, 80, 88, 96]


def test_every_read_is_bounded(kernels):
    for ranks, body in kernels:
        loads = re.findall(r"^\s+((?:global|flat|buffer|scratch)_load\w+)", body, re.M)
        assert set(loads) == {"buffer_load_dwordx4"}, f"{ranks} ranks: {sorted(set(loads))}"
        # eight rows of the other operand, and a fragment of 16 ranks each
        assert len(loads) >= 8 + ranks // 16
