"""Host arithmetic of the rows' kernels (csrc/rows8.hpp), compiled for the host."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "rows8.hpp"
extern "C" void rows_of_part(int64_t rows, int parts, int part, int64_t* first, int64_t* last) {
    const sfm::RowRange r = sfm::rows_of_part(rows, parts, part);
    *first = r.first;
    *last = r.last;
}
extern "C" void wide_grid(int64_t wgs, unsigned* x, unsigned* y) {
    const dim3 g = sfm::wide_grid(wgs);
    *x = g.x;
    *y = g.y;
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.hip").write_text(SOURCE)
    csrc = os.path.join(ROOT, "self-forcing_amd", "csrc")
    subprocess.run([hipcc, "--offload-host-only", "-std=c++17", "-shared", "-fPIC", "-I" + csrc, "-I" + os.path.join(ROOT, "include"),
                    str(d / "rules.hip"), "-o", str(d / "rules.so")], check=True, capture_output=True)
    return C.CDLL(str(d / "rules.so"))


@pytest.mark.parametrize("rows", [1, 3, 4, 1560, 32760, 2 ** 31 - 769, 2 ** 31 - 768, 2 ** 31 - 1])
@pytest.mark.parametrize("parts", [1, 2, 25, 512, 768])
def test_the_parts_of_a_group_are_its_rows_once(rules, rows, parts):
    at = 0
    for part in range(parts):
        first, last = C.c_int64(0), C.c_int64(0)
        rules.rows_of_part(C.c_int64(rows), parts, part, C.byref(first), C.byref(last))
        if first.value < last.value:
            assert first.value == at and last.value <= rows
            at = last.value
        else:
            assert at == rows                                   # nothing is left
    assert at == rows


@pytest.mark.parametrize("wgs", [1, 2, 4680, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, 23200 * 23200 // 32, 2 ** 31])
def test_grids_stay_within_what_the_runtime_takes(rules, wgs):
    x, y = C.c_uint(0), C.c_uint(0)
    rules.wide_grid(C.c_int64(wgs), C.byref(x), C.byref(y))
    assert x.value * 1024 < 2 ** 32 and y.value * 1024 < 2 ** 32
    assert wgs <= x.value * y.value < wgs + x.value
    assert wgs > 2 ** 21 or y.value == 1
