"""What the compiler makes of device code, seen in the assembly of small kernels built for gfx950 (no GPU needed)."""
import os
import re
import subprocess

import pytest

from face_recognition_amd import build

TWO_USERS_OF_M0 = """
#include "pj_tile.h"
using namespace fra;
__global__ void two_users(const float* g, float* out) {
    __shared__ __attribute__((aligned(16))) char lds[4096];
    typedef __attribute__((address_space(3))) void* P;
    __builtin_amdgcn_global_load_lds(g + threadIdx.x * 4, (P)((LdsPtr)lds + 1024), 16, 0, 0);
    dma16(g + 1024 + threadIdx.x * 4, (LdsPtr)lds + 2048);
    __builtin_amdgcn_global_load_lds(g + 2048 + threadIdx.x * 4, (P)((LdsPtr)lds + 1024), 16, 0, 0);
    dma_wait_barrier<0>();
    out[threadIdx.x] = reinterpret_cast<const float*>(lds)[threadIdx.x];
}
"""


def test_dma16_names_the_register_it_sets(tmp_path):
    """A load into LDS takes its address from m0.  The compiler sets m0 for its own such loads, here twice to the same value: the
    second must not rely on the first's setting, which dma16 between them has overwritten."""
    try:
        hipcc = build._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    src, asm = tmp_path / "m0.hip", tmp_path / "m0.s"
    src.write_text(TWO_USERS_OF_M0)
    r = subprocess.run([hipcc, "-O3", "-std=c++17", f"--offload-arch={build.ARCH}", "--cuda-device-only", "-S", "-x", "hip", "-I", build.CSRC,
                        "-I", os.path.join(build.HERE, "..", "include"), str(src), "-o", str(asm)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    # per load: whether m0 was written since the load before it
    fresh, written = [], False
    for line in asm.read_text().splitlines():
        if re.match(r"\s*s_\w+ m0,", line):
            written = True
        elif "global_load_lds" in line:
            fresh.append(written)
            written = False
    assert fresh == [True, True, True]
