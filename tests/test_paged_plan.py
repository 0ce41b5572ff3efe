"""The plans of vva_paged_attn over few rows count on no more workgroups at once than fit: the piece of a sequence that a
workgroup beyond them takes waits for a second round.  What fits goes by the registers and the LDS of the compiled kernels,
from the notes of their code object."""
import os
import re
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJ = os.path.join(REPO, "vibevoice.cpp_amd", "obj", "paged_attn.hip.o")
PLAN = os.path.join(REPO, "tests", "cpp", "bin", "paged_plan")
LLVM = "/opt/rocm/llvm/bin"
CUS, LDS, VGPRS = 256, 160 * 1024, 512             # of the GPU; bytes of a CU; of a SIMD's lane, 4 SIMDs a CU
Q8_0 = 8


@pytest.fixture(scope="module")
def fits(tmp_path_factory):
    """(page type, head dim, waves of a workgroup) -> workgroups of a CU, the fewest of the result types."""
    if not (os.path.exists(OBJ) and os.path.exists(os.path.join(LLVM, "clang-offload-bundler"))):
        pytest.skip("no object file of the kernels here, or no ROCm LLVM")
    at = tmp_path_factory.mktemp("co")
    fat, co = str(at / "fat"), str(at / "co")
    subprocess.run([f"{LLVM}/llvm-objcopy", f"--dump-section=.hip_fatbin={fat}", OBJ, str(at / "o")], check=True)
    subprocess.run([f"{LLVM}/clang-offload-bundler", "--unbundle", "--type=o", f"--input={fat}", f"--output={co}",
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950"], check=True)
    notes = subprocess.run([f"{LLVM}/llvm-readelf", "--notes", co], capture_output=True, text=True, check=True).stdout
    got = {}
    for k in notes.split("  - .agpr_count:")[1:]:
        name = re.search(r"\.name:\s+(\S+)", k).group(1)
        m = re.search(r"paged_few_kernelILi(\d+)ELi(\d+)ELi\d+ELi(\d+)ELi\d+E", name)
        if not m:
            continue
        d, page_type, waves = map(int, m.groups())
        vgprs, lds = (int(re.search(rf"\.{x}:\s+(\d+)", k).group(1)) for x in ("vgpr_count", "group_segment_fixed_size"))
        of_simd = min(8, VGPRS // (-(-vgprs // 8) * 8))
        n = min(4 * of_simd // waves, LDS // lds)
        got[page_type, d, waves] = min(n, got.get((page_type, d, waves), n))
    assert len(got) == 8, got
    return got


def test_pieces_of_few_rows_run_at_once(fits):
    if not os.path.exists(PLAN):
        pytest.fail("tests/cpp not built: run __graft_entry__.build()")
    lines = subprocess.run([PLAN], capture_output=True, text=True, check=True).stdout.splitlines()
    assert len(lines) > 300
    over = []
    for line in lines:
        t, d, hq, hkv, rows, n_seq, waves, wgs = map(int, line.split())
        assert waves == (8 if t == Q8_0 and rows <= 16 else 4), line
        if wgs > CUS * fits[t, d, waves]:
            over.append((line, fits[t, d, waves]))
    assert not over, over
