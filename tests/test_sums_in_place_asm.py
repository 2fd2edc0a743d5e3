"""Matrix instructions written as assembly, whose waits the compiler does not know: the sums of a loop are touched by nothing before the wait behind
it, and a loop with so few sums that one comes up again too early does not compile."""
import re
import subprocess

import pytest

from oztt_amd import build as B

FILES = {"oz_linear_tiles.hip": 6, "oz_linear_i8.hip": 2, "oz_newton_schulz.hip": 10, "oz_newton_schulz_three.hip": 5}
ACCUMULATORS = re.compile(r"\ba(\d+)\b|\ba\[(\d+):(\d+)\]")


def registers(line):
    out = set()
    for one, first, last in ACCUMULATORS.findall(line):
        out |= {int(one)} if one else set(range(int(first), int(last) + 1))
    return out


def code(text):
    """(line, whether it was written as assembly)"""
    out, written = [], False
    for l in text.split("\n"):
        if "#ASMSTART" in l or "#ASMEND" in l:
            written = "#ASMSTART" in l
            continue
        l = l.split(";")[0].strip()
        if l and (not l.startswith(".") or l.startswith(".LBB")):
            out.append((l, written))
    return out


def unsettled(lines, start):
    """The instructions that may run behind the one at `start` before a wait does."""
    labels = {l[:-1]: i for i, (l, _) in enumerate(lines) if l.endswith(":")}
    seen, ways = set(), [start + 1]
    while ways:
        i = ways.pop()
        while i not in seen and not (lines[i][0] == "s_nop 15" and lines[i + 1][0] == "s_nop 15"):
            seen.add(i)
            l = lines[i][0]
            assert not l.startswith(("s_setpc", "s_endpgm")), "an end without a wait"
            if m := re.match(r"s_c?branch\S*\s+(\S+)$", l):
                ways.append(labels[m.group(1)])
                if l.startswith("s_branch"):
                    break
            i += 1
    return seen


@pytest.mark.parametrize("src", sorted(FILES))
def test_nothing_touches_a_sum_before_the_wait(src, tmp_path):
    r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, *B.HIP_SOURCES[src], "--cuda-device-only", "-S", str(B.CSRC / src), "-o", str(tmp_path / "x.s")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    loops = 0
    for kernel, text in re.findall(r"\n(_Z\S*kernel\S*):(.*?)\.Lfunc_end", (tmp_path / "x.s").read_text(), re.S):
        lines = code(text)
        left = {i for i, (l, written) in enumerate(lines) if written and l.startswith("v_mfma")}
        while left:
            after = unsettled(lines, min(left))
            mine = left & after | {min(left)}
            sums = set().union(*(registers(lines[i][0]) for i in mine))
            assert len(sums) >= 64, kernel
            touched = [lines[i][0] for i in sorted(after - mine) if registers(lines[i][0]) & sums]
            assert not touched, (kernel, touched[:4])
            left -= mine
            loops += 1
    assert loops == FILES[src], loops


@pytest.mark.parametrize("blocks,compiles", [(8, True), (4, True), (2, False)])
def test_least_sums(blocks, compiles, tmp_path):
    (tmp_path / "x.hip").write_text('#include "oz_linear_tiles.hpp"\ntemplate struct ozl::BigLoop<ozt::Half<OZ_F16>, false, false, %d>;\n' % blocks)
    r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, "--cuda-device-only", "-fsyntax-only", str(tmp_path / "x.hip")], capture_output=True, text=True)
    assert (r.returncode == 0) == compiles, r.stderr[-2000:]
    assert compiles or "distance of a sum's instructions" in r.stderr
