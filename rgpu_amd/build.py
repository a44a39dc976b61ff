"""Build librtensor_hip.so (gfx950) in-tree from rgpu_amd/csrc.

    python -m rgpu_amd.build          # or rgpu_amd.build.build()

Every source is compiled with hipcc for --offload-arch=gfx950 into
rgpu_amd/_build/*.o and linked into rgpu_amd/librtensor_hip.so, which the
ctypes bindings in rgpu_amd/gpu.py load.  Sources whose arithmetic must round
like rtensor's CPU path (optimizer, row kernels) get -ffp-contract=off.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "librtensor_hip.so")
ARCH = "gfx950"

SOURCES = {
    "runtime.hip": [],
    "mlp.hip": [],
    "gemm_f32.hip": [],
    "gemm_half.hip": [],
    "rowops.hip": ["-ffp-contract=off"],
    "optim.hip": ["-ffp-contract=off"],
    "tensor_ops.hip": ["-ffp-contract=off"],
    "noalloc.hip": [],
    "mx.hip": [],
    "mx_gemm.hip": [],
    "mx_backward.hip": [],
}

COMMON = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-Wall", "-Wno-unused-function", "-Wno-unused-value", "-Wno-unused-result",
    # Keep the compiler from forming packed-FP32 (v_pk_*_f32) instructions.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I", os.path.join(ROOT, "include"), "-I", CSRC,
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found")


def _compile(src: str, extra) -> str:
    obj = os.path.join(OUT, os.path.splitext(src)[0] + ".o")
    cmd = [hipcc(), *COMMON, *extra, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    err = "\n".join(l for l in (r.stderr or "").splitlines() if "packed-fp32-ops" not in l)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{err}")
    if err.strip():
        sys.stderr.write(err + "\n")
    return obj


def build(jobs: int = 6) -> str:
    """Compile every source and link the shared library; returns its path."""
    os.makedirs(OUT, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=max(1, min(jobs, len(SOURCES)))) as ex:
        objs = list(ex.map(lambda kv: _compile(*kv), SOURCES.items()))
    tmp = LIB + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stderr)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build())
