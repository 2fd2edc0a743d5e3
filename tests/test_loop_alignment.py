"""Loops of the linear layers' tiles begin at whole lines of the instruction cache."""
import re
import subprocess

from oztt_amd import build as B


def test_loops_with_matrix_instructions(tmp_path):
    src = "oz_linear_tiles.hip"
    r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, *B.HIP_SOURCES[src], "--cuda-device-only", "-S", str(B.CSRC / src), "-o", str(tmp_path / "x.s")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    loops = 0
    for kernel, text in re.findall(r"\n(_Z\S*product_\S*kernel\S*):(.*?)\.Lfunc_end", (tmp_path / "x.s").read_text(), re.S):
        lines = [l for l in text.split("\n") if l.strip() and not l.strip().startswith(";")]
        found = 0
        for i, l in enumerate(lines):
            m = re.match(r"(\.LBB\d+_\d+):.*Loop Header: Depth=1", l)
            if m:
                ends = [k for k in range(i, len(lines)) if re.search(r"s_c?branch\S*\s+%s$" % re.escape(m.group(1)), lines[k].strip())]
                if ends and any("v_mfma" in x for x in lines[i : ends[-1]]):
                    assert re.match(r"\.p2align\s+6\b", lines[i - 1].strip()), (kernel, l, lines[i - 1])
                    found += 1
        assert found == 1, (kernel, found)
        loops += found
    assert loops == 30, loops
