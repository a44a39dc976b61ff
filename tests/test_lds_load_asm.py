"""The wait state between a write of M0 and a load into LDS (no GPU needed: hipcc compiles the helpers here).

gfx950 takes the LDS destination of a direct-to-LDS load from M0, and wants one wait state after a scalar instruction that
wrote it.  The compiler keeps it for its own loads; it does not look into inline asm, so rt_dev's asm helpers have to."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "rgpu_amd", "csrc")

HELPERS = {
    "dma16": "rt_dev::dma16(r, smem + 1024 * i, voff, 64 * i)",
    "dma16_asm": "rt_dev::dma16_asm(r, smem + 1024 * i, voff, 64 * i)",
    "dma16_at": "rt_dev::dma16_at(r, rt_dev::lds_offset(smem) + 1024 * i, voff)",
    "dma4_at": "rt_dev::dma4_at(r, rt_dev::lds_offset(smem) + 1024 * i, voff)",
}
PROBE = """
#include "device_util.h"
__global__ void probe(const char* p, float* out, int bytes) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[4096];
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, bytes, 0x00020000);
  const int voff = 16 * threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) CALL;
  rt_dev::wait_vm<0>();
  rt_dev::barrier_lds();
  out[threadIdx.x] = reinterpret_cast<float*>(smem)[threadIdx.x];
}
"""


def instructions(text):
    """What is executed, in order: comments and directives left out, an encoded s_nop under its name."""
    out = []
    for line in text.split("\n"):
        line = line.split(";")[0].strip()
        if re.fullmatch(r"\.long\s+0xbf80000[0-9a-f]", line):
            line = "s_nop %d" % int(line[-1], 16)
        if line and not line.startswith(".") and not line.endswith(":"):
            out.append(line)
    return out


@pytest.mark.parametrize("helper", sorted(HELPERS))
def test_a_load_into_lds_waits_for_m0(helper, tmp_path):
    hipcc = next((c for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc")
                  if c and os.path.exists(c)), None)
    if hipcc is None:
        pytest.skip("hipcc not available")
    src, asm = tmp_path / "probe.hip", tmp_path / "probe.s"
    src.write_text(PROBE.replace("CALL", HELPERS[helper]))
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-I", CSRC, "-S", "--cuda-device-only",
                        str(src), "-o", str(asm)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    code = instructions(asm.read_text())
    loads = [i for i, l in enumerate(code) if l.startswith("buffer_load") and l.endswith(" lds")]
    assert len(loads) == 4
    for i in loads:
        before = code[i - 1]
        assert not re.search(r"\bm0\b", before), (before, code[i])


def test_no_other_asm_loads_into_lds():
    """The helpers above are the only inline asm that does."""
    for name in sorted(os.listdir(CSRC)):
        text = open(os.path.join(CSRC, name)).read()
        found = re.findall(r'"[^"\n]*buffer_load[^"\n]*lds[^"\n]*"', text)
        assert len(found) == (3 if name == "device_util.h" else 0), (name, found)
