"""The code generated for the products that copy operands into LDS by inline asm (oz_linear_tiles.hip): M0, which a copy sets
itself, serves nothing else; nothing spills (scratch accesses would enter the counts that the copies' waits rely on); the large
tile's loop moves no sums between registers."""
import re
import subprocess

import pytest

from oztt_amd import build as B


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "x.s"
    src = "oz_linear_tiles.hip"
    cmd = [B.HIPCC, *B.HIP_FLAGS, *B.HIP_SOURCES[src], "--cuda-device-only", "-S", str(B.CSRC / src), "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return out.read_text()


def test_m0_and_spills(asm):
    body = [x for x in (l.strip() for l in asm.split("\n")) if x and not x.startswith(";")]
    m0 = [i for i, l in enumerate(body) if re.search(r"\bm0\b", l) and not l.startswith(".")]
    assert m0 and all(re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi|ttmp\d+)$", body[i]) for i in m0)
    assert all(body[i + 1] == "s_nop 0" and re.match(r"buffer_load_dwordx4 .* offen lds$", body[i + 2]) for i in m0)
    assert sum(l.startswith("buffer_load") for l in body) == len(m0)
    meta = re.findall(r"\.name:\s+(_Z\S*product_\S*)\s.*?\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", asm, re.S)
    assert len(meta) == 30 and all(p == "0" and s == "0" for _, p, s in meta), meta


def test_the_large_tile_keeps_its_sums_in_place(asm):
    kernels = re.findall(r"\n(_ZN3ozl18product_big_kernel\S*):(.*?)\.Lfunc_end", asm, re.S)
    assert len(kernels) == 6
    for name, text in kernels:
        blocks = [b for b in re.split(r"\n\.LBB", text) if "v_mfma" in b]
        assert sum(b.count("v_mfma") for b in blocks) == 128, name  # two steps of 64, unrolled no further
        assert not any("v_accvgpr" in b or "scratch_" in b for b in blocks), name
