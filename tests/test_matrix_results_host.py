"""Matrix instructions that stand in inline assembly: the compiler knows nothing
of the time their results take, so no other instruction, copies that it adds by
itself included, may read one before it is there.  Checked in the assembly of every
kernel that has such instructions, along all branches."""

import concurrent.futures
import re
import subprocess

import pytest

from eth_amd import build as eb

# a 16x16x32 instruction (8 passes) is read 11 wait states behind it, at the earliest
NEEDED = 12
SOURCES = ("gemm", "linear_xent", "adapters")


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm")

    def compile_one(name):
        path = out / f"{name}.s"
        subprocess.run([eb.hipcc_path(), *eb.HIPCC_FLAGS, f"-I{eb.INCLUDE}", "--cuda-device-only", "-S",
                        str(eb.CSRC / f"{name}.hip"), "-o", str(path)], check=True, capture_output=True, timeout=300)
        return path.read_text()

    with concurrent.futures.ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        return dict(zip(SOURCES, pool.map(compile_one, SOURCES)))


def _registers(text):
    got = set()
    for one, n, many, a, b in re.findall(r"\b([av])(\d+)\b|\b([av])\[(\d+):(\d+)\]", text):
        got |= {(one, int(n))} if one else {(many, i) for i in range(int(a), int(b) + 1)}
    return got


def _kernels(text):
    """(name, [(instruction, whether in inline assembly)], label -> place)"""
    for m in re.finditer(r"^(_Z\w+):.*?\n(.*?)^\.Lfunc_end", text, re.M | re.S):
        lines, labels, inline = [], {}, False
        for line in m.group(2).splitlines():
            if "#ASMSTART" in line or "#ASMEND" in line:
                inline = "#ASMSTART" in line
                continue
            line = re.sub(r";.*", "", line).strip()
            if re.match(r"\.LBB\w+:", line):
                labels[line[:-1]] = len(lines)
            elif line and not line.startswith("."):
                lines.append((line, inline))
        yield m.group(1), lines, labels


def early_reads(lines, labels):
    """(matrix instruction, reader) pairs less than NEEDED wait states apart."""
    found = []
    for i, (line, inline) in enumerate(lines):
        if not (inline and line.startswith("v_mfma")):
            continue
        result = _registers(line.split(None, 1)[1].split(",")[0])
        todo, best = [(i + 1, 0)], {}
        while todo:
            j, waited = todo.pop()
            while j < len(lines) and waited < NEEDED and best.get(j, NEEDED) > waited:
                best[j] = waited
                other, _ = lines[j]
                name = other.split()[0]
                if name == "s_endpgm":
                    break
                if name == "s_nop":
                    waited += int(other.split()[1], 0)
                elif "branch" in name:
                    todo.append((labels[other.split()[1]], waited + 1))
                    if name == "s_branch":
                        break
                elif name.startswith("v_mfma"):
                    # as an accumulator it is passed on; as a factor it is read
                    factors = re.split(r",\s*(?![^\[]*\])", other.split(None, 1)[1])[1:3]
                    if _registers(",".join(factors)) & result:
                        found.append((line, other))
                elif _registers(other) & result:
                    found.append((line, other))
                    break
                waited += 1
                j += 1
    return found


def test_the_check_finds_an_early_read():
    mfma = ("v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]", True)
    copy = ("v_accvgpr_write_b32 a0, v3", False)
    assert early_reads([mfma, ("s_nop 7", False), copy], {}) and not early_reads([mfma, ("s_nop 15", False), copy], {})
    loop = [("v_add_f32_e32 v9, v2, v9", False), mfma, ("s_cbranch_vccnz .LBB0_1", False), ("s_endpgm", False)]
    assert early_reads(loop, {".LBB0_1": 0}) and not early_reads(loop, {".LBB0_1": 3})
    assert not early_reads([mfma, mfma, ("s_endpgm", False)], {})


@pytest.mark.parametrize("source", SOURCES)
def test_no_result_is_read_early(assembly, source):
    checked = 0
    for name, lines, labels in _kernels(assembly[source]):
        if any(inline and line.startswith("v_mfma") for line, inline in lines):
            checked += 1
            assert not early_reads(lines, labels), name
    assert checked >= 8
