"""The direct global-to-LDS load's instruction sequence (cxm_common.hpp), from
the assembly of a small kernel built here: its scalar base is written by the
scalar unit in the instruction before.  A vector-memory instruction may read an
SGPR written by a vector instruction only five wait states later (and M0 one
after its write), and the compiler does not look into asm for that."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

SOURCE = """
#include "cxm_common.hpp"
using namespace cxm;
__global__ void k(const char *x, const unsigned *at, float *out) {
    __shared__ __attribute__((aligned(16))) float s[512];
    // a base that the vector unit computes, and one that the scalar unit does
    lds_load16_at(x + at[threadIdx.x / 64] * 64ul, threadIdx.x % 64 * 16, lds_addr(s));
    lds_load16_at(x + blockIdx.x * 1024ul, threadIdx.x % 64 * 16, lds_addr(s + 256));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    out[threadIdx.x] = s[threadIdx.x] + s[threadIdx.x + 256];
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_base_of_direct_loads_is_scalar_written(tmp_path):
    src, asm = tmp_path / "k.hip", tmp_path / "k.s"
    src.write_text(SOURCE)
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "--offload-device-only", "-S",
                    "-I", os.path.join(ROOT, "cortexmind_amd", "csrc"), str(src), "-o", str(asm)], check=True,
                   capture_output=True)
    lines = [l.strip() for l in asm.read_text().splitlines()]
    code = [l for l in lines if l and not l.startswith((";", ".")) and not l.endswith(":")]
    loads = [i for i, l in enumerate(code) if l.startswith("global_load_lds_dwordx4")]
    assert len(loads) == 2
    for i in loads:
        base = re.search(r"s\[\d+:\d+\]", code[i]).group()
        assert re.match(r"s_mov_b64 " + re.escape(base) + ",", code[i - 1]), code[i - 1:i + 1]
