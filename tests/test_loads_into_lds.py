"""The inline form of a load into LDS beside the compiler's own, from the assembly of a kernel that has both.  Needs no GPU."""
import re
import subprocess

from cats_amd.build import HIP_FLAGS, HIPCC

SOURCE = """
#include <hip/hip_runtime.h>
#include "cats_packed.h"
namespace cats {
__device__ __forceinline__ void bring(const char* from, char* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + threadIdx.x * 16), (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
__global__ void both(const char* a, const char* b, const char* c, float* out) {
  __shared__ __align__(16) char s[3][1024];
  bring(a, s[1]);
  load_lds(b, threadIdx.x * 16, s[2]);
  bring(c, s[1]);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  out[threadIdx.x] = ((float*)s)[threadIdx.x * 8];
}
}
"""


def test_the_compiler_s_loads_have_their_own_address_behind_an_inline_one(tmp_path):
    """Where a load goes is in m0.  Two to one place, with an inline one to another place between them: m0 is set before each of the three."""
    source, out = tmp_path / "both.hip", tmp_path / "both.s"
    source.write_text(SOURCE)
    subprocess.run([HIPCC, *HIP_FLAGS, "--cuda-device-only", "-S", str(source), "-o", str(out)], check=True, capture_output=True)
    lines = [m[0] for m in re.finditer(r"^\s+(\w+ m0,|global_load_lds_dwordx4).*$", out.read_text(), re.M)]
    loads = [i for i, line in enumerate(lines) if "global_load" in line]
    assert len(loads) == 3 and all(i > 0 and "m0," in lines[i - 1] for i in loads), lines
