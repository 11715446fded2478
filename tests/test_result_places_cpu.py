"""Host-side checks of where a result may lie (csrc/matrix.hpp): exactly in its input's place, but not
where other results read the same memory."""
import os
import subprocess

import pytest

from conftest import REPO

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
PROBE = r"""
#include <stdio.h>
#include "matrix.hpp"
namespace ttpi {
int fail(int code, const std::string& m) { return printf("%s\n", m.c_str()), code; }
int device_buffer(const ttp_ctx*, const void*, uint64_t, const char*, SeenAlloc*) { return 0; }
}
int main() {
    static float memory[64];
    const ttp_matrix m{memory, 8, 8, 8, TTP_DTYPE_F32, 0}, row{memory, 1, 8, 8, TTP_DTYPE_F32, 0};
    for (int shared = 0; shared < 2; ++shared) {  // x and the residual, of which y may be one
        ttpi::Buffers b(nullptr);
        b.matrix(&m, 8, 8, "x", false, nullptr, shared);
        b.matrix(&m, 8, 8, "residual", false);
        printf("%d\n", b.matrix(&m, 8, 8, "y", true, &m));
    }
    for (int own = 0; own < 2; ++own) {  // a row in the place of an input that is an array, too
        ttpi::Buffers b(nullptr);
        b.matrix(&row, 1, 8, "x", false);
        own ? b.own(memory, 8, 4, "array", false) : b.array(memory, 8, 4, "array", false);
        printf("%d\n", b.matrix(&row, 1, 8, "y", true, &row));
    }
}
"""


def test_a_result_in_the_place_of_several_inputs(tmp_path):
    if not os.path.exists(os.path.join(ROCM, "include", "hip", "hip_runtime.h")):
        pytest.skip("HIP's headers absent")
    (tmp_path / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I",
                    os.path.join(ROCM, "include"), "-I", os.path.join(REPO, "include"), "-I",
                    os.path.join(REPO, "tt-perf_amd", "csrc"), "-o", str(tmp_path / "probe"),
                    str(tmp_path / "probe.cpp")], check=True, capture_output=True)
    out = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout
    assert out.splitlines() == ["0", "y overlaps x", "-1", "y overlaps array", "-1",
                                "y overlaps array", "-1"]
