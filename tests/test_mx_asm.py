"""The assembly of the microscaled product (no GPU needed: hipcc compiles it here).

The rows of C go through LDS between the lanes of one wave without a workgroup barrier: every read there has to stay behind
the writes before it, and the next writes behind the reads, which the wave barriers see to."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "rgpu_amd", "csrc")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    hipcc = next((c for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc")
                  if c and os.path.exists(c)), None)
    if hipcc is None:
        pytest.skip("hipcc not available")
    out = str(tmp_path_factory.mktemp("asm") / "mx_gemm.s")
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                        "-packed-fp32-ops", "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-S", "--cuda-device-only",
                        os.path.join(CSRC, "mx_gemm.hip"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return open(out).read()


def test_lanes_that_pass_rows_through_lds_are_ordered(asm):
    names = re.findall(r"^(_Z\w*mx_gemm_kernel\w*):", asm, re.M)
    assert len(names) == 5
    for name in names:
        bm, wgm = (int(v) for v in re.search(r"ILi\dELi(\d+)ELi\d+ELi(\d)E", name).groups())
        body = asm[asm.index(name + ":"):]
        written, barriers = False, 0
        for line in body[:body.index(".Lfunc_end")].split("\n"):
            line = line.strip()
            if line.startswith(("; wave barrier", "s_barrier")):
                written, barriers = False, barriers + line.startswith(";")
            elif line.startswith("ds_write"):
                written = True
            elif line.startswith("ds_read"):
                assert not written, (name, line)
        # two output types; 16 rows a turn: one before each turn's reads, one before each but the first one's writes
        assert barriers == 2 * (2 * (bm // wgm // 16) - 1), name
