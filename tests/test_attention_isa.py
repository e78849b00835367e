"""CPU: the registers of attention's forward instances, as the compiler reports them: what only the position table's form needs is in no other instance."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"
# head size, waves along the queries / the keys, table; the vector registers that may go through memory (a tile's loop at 128 keeps 200 of 256 in operands
# and results: a few addresses leave them)
FORMS = [(64, 4, 1, False, 0), (96, 4, 1, False, 0), (96, 4, 1, True, 0), (96, 1, 2, False, 0), (128, 4, 1, False, 16), (128, 4, 1, True, 16), (128, 1, 2, False, 0)]


@pytest.fixture(scope="module")
def spills(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("needs hipcc")
    d = tmp_path_factory.mktemp("isa")
    src = '#include "attn_fwd.inc"\nnamespace attn {\n' + "".join(
        f"template __global__ void fwd_k<re_bf16, {D}, {wq}, {wk}, true, true, {str(table).lower()}>(const args, const fwd_out);\n" for D, wq, wk, table, _ in FORMS) + "}\n"
    (d / "forms.hip").write_text(src)
    subprocess.run([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S",
                    "-I" + os.path.join(ROOT, "recboard_amd", "csrc"), str(d / "forms.hip"), "-o", str(d / "forms.s")], check=True, capture_output=True)
    found = re.findall(r"\.name:\s+\S*fwd_kIDF16bLi(\d+)ELi(\d)ELi(\d)ELb1ELb1ELb(\d)E.*?\.vgpr_spill_count:\s+(\d+)", (d / "forms.s").read_text(), re.S)
    return {(int(D), int(wq), int(wk), t == "1"): int(n) for D, wq, wk, t, n in found}


@pytest.mark.parametrize("D,wq,wk,table,most", FORMS)
def test_aligned_forms_with_a_mask_or_a_table_keep_their_registers(spills, D, wq, wk, table, most):
    assert spills[D, wq, wk, table] <= most


def test_inline_assembly_that_writes_m0_says_so():
    """A loader of LDS addresses its destination through m0; the compiler may keep a value of its own there unless the statement names it."""
    wrote = 0
    for name in sorted(os.listdir(os.path.join(ROOT, "recboard_amd", "csrc"))):
        if not name.endswith((".h", ".inc", ".hip")):
            continue
        with open(os.path.join(ROOT, "recboard_amd", "csrc", name)) as f:
            src = f.read()
        for m in re.finditer(r'asm volatile\((.*?)\);', src, re.S):
            if re.search(r"\bs_\w+ m0,", m.group(1)):
                wrote += 1
                assert '"m0"' in m.group(1).rsplit(":", 1)[1], (name, m.group(0))
    assert wrote
