"""CPU: which strides attention's aligned form takes.  Its tiles are loaded by 32-bit unsigned byte offsets from their first row, so rows have to follow each
other upwards, and not too far apart; everything else goes to the form that computes 64-bit addresses element by element.  The rule is
compiled from the kernels' own header and asked here; nothing is launched."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ASK = r"""
#include "attn_common.h"
#include <cstdio>
#include <cstdlib>
// dtype, D, then (pointer offset, batch, head, row) stride; prints the answer for that tensor beside an ordinary one
int main(int n, char** v) {
    const int32_t dtype = atoi(v[1]);
    attn::args a{};
    a.D = atoi(v[2]);
    for (int i = 3; i + 3 < n; i += 4) {
        const int64_t ordinary[3] = {1 << 20, 1 << 16, 128}, s[3] = {atoll(v[i + 1]), atoll(v[i + 2]), atoll(v[i + 3])};
        printf("%d", (int)attn_aligned(a, dtype, {{(void*)4096, ordinary}, {(char*)4096 + atoi(v[i]), s}, {(void*)8192, ordinary}}));
    }
}
"""
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    if not shutil.which(HIPCC):
        pytest.skip("needs hipcc")
    d = tmp_path_factory.mktemp("ask")
    (d / "ask.hip").write_text(ASK)
    subprocess.run([HIPCC, "-std=c++17", "--offload-host-only", "-Wno-unused-function", "-I" + os.path.join(ROOT, "recboard_amd", "csrc"), str(d / "ask.hip"),
                    "-o", str(d / "ask")], check=True)

    def run(dtype, D, *tensors):
        out = subprocess.run([str(d / "ask"), str(dtype), str(D)] + [str(x) for t in tensors for x in t], check=True, capture_output=True, text=True).stdout
        return [c == "1" for c in out]
    return run


@pytest.mark.parametrize("dtype,D", [(0, 64), (1, 64), (2, 128)])
def test_rows_that_go_backwards_are_not_loaded_by_unsigned_offsets(ask, dtype, D):
    up = (0, 1 << 20, 1 << 16, D)
    down = [(0, 1 << 20, 1 << 16, -D), (0, 0, 0, -8), (0, 1 << 20, 1 << 16, -(1 << 22)), (0, 1 << 20, 1 << 16, -(1 << 40))]
    assert ask(dtype, D, up, *down) == [True] + [False] * 4


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_the_other_strides(ask, dtype):
    """Batches and heads may go any way (their offsets are 64 bits wide); rows may stand still or lie up to 2^22 elements apart; everything on 16 bytes."""
    yes = [(0, -(1 << 40), -(1 << 33), 64), (0, 0, 0, 0), (0, 8, 8, 1 << 22), (16, 64, 64, 64)]
    no = [(0, 8, 8, (1 << 22) + 8), (0, 8, 8, 1 << 33), (2, 8, 8, 64), (0, 8, 8, 66 if dtype else 65), (0, 7, 8, 64), (0, 8, -7, 64)]
    assert ask(dtype, 64, *yes, *no) == [True] * len(yes) + [False] * len(no)
    assert ask(dtype, 63, yes[0]) == [False]
