"""The code generated for the operators on weights whose products copy operands into LDS by inline asm: M0, which a copy sets itself, serves
nothing else; nothing spills (scratch accesses would enter the counts that the copies' waits rely on); loops with sums in accumulation
registers leave them in place."""
import re
import subprocess

import pytest

from oztt_amd import build as B

FILES = {"oz_linear_i8.hip": (10, "scaled_(?:tile|big)_kernel"), "oz_newton_schulz.hip": (9, "newton_schulz_kernel"), "oz_newton_schulz_three.hip": (6, "newton_schulz_kernel")}


@pytest.fixture(scope="module", params=sorted(FILES))
def built(request, tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "x.s"
    src = request.param
    cmd = [B.HIPCC, *B.HIP_FLAGS, *B.HIP_SOURCES[src], "--cuda-device-only", "-S", str(B.CSRC / src), "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return src, out.read_text()


def test_m0_and_spills(built):
    src, asm = built
    count, name = FILES[src]
    body = [x for x in (l.strip() for l in asm.split("\n")) if x and not x.startswith(";")]
    m0 = [i for i, l in enumerate(body) if re.search(r"\bm0\b", l) and not l.startswith(".")]
    assert m0 and all(re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi|ttmp\d+)$", body[i]) for i in m0)
    assert all(body[i + 1] == "s_nop 0" and re.match(r"buffer_load_dwordx4 v\d+, s\[\d+:\d+\], 0 offen lds$", body[i + 2]) for i in m0)
    assert sum(l.startswith("buffer_load") for l in body) == len(m0)
    meta = re.findall(r"\.name:\s+(_Z\S*(?:%s)\S*)\s.*?\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)" % name, asm, re.S)
    assert len(meta) == count and all(p == "0" and s == "0" for _, p, s in meta), meta


def test_streams_do_not_spill(built):
    src, asm = built
    if src != "oz_linear_i8.hip":
        return
    meta = re.findall(r"\.name:\s+(_Z\S*(?:stream|few_rows)_kernel\S*)\s.*?\.private_segment_fixed_size:\s+(\d+)", asm, re.S)
    assert len(meta) == 9 and all(p == "0" for _, p in meta), meta


def test_sums_stay_in_place(built):
    """Innermost loops with 32 matrix instructions or more."""
    src, asm = built
    found = 0
    for kernel, text in re.findall(r"\n(_Z\S*(?:%s)\S*):(.*?)\.Lfunc_end" % FILES[src][1], asm, re.S):
        lines, labels = text.split("\n"), {}
        for i, l in enumerate(lines):
            if m := re.match(r"(\.LBB\d+_\d+):", l):
                labels[m.group(1)] = i
            m = re.search(r"s_c?branch\S*\s+(\.LBB\d+_\d+)", l)
            if m and m.group(1) in labels:
                loop = lines[labels[m.group(1)] : i + 1]
                if sum("v_mfma" in x for x in loop) >= 32:
                    found += 1
                    assert not any("v_accvgpr" in x or "scratch_" in x for x in loop), kernel
    assert found >= {"oz_linear_i8.hip": 2, "oz_newton_schulz.hip": 10, "oz_newton_schulz_three.hip": 5}[src], found
