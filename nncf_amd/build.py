"""Builds libnncf_amd_wc.so (HIP kernels + C ABI) in-tree for gfx950 with hipcc.

    python -m nncf_amd.build [--force]

Cross-compiles without a GPU.  -ffp-contract=off is REQUIRED: bit-exact parity with the reference needs
separately rounded fp32 divide/add (see csrc/wc_common.h).
"""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libnncf_amd_wc.so")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fno-fast-math",
         "-Wall", "-Wno-unused-function", "-Wno-inline-asm"]
# per-file additions.  wc_cholinv.hip: the SLP vectoriser pairs the rank-16 updates of the panel kernel into v_pk_fma_f32
# and pays for it with ~2300 register moves and 110 more registers (15 000 -> 13 300 instructions per wave without it)
# wc_linear*.hip, wc_gemm_*.hip, wc_experts.hip: no packed fp32 instructions, some of whose forms are not dependable on this
# hardware (the host pass does not know the feature and says so)
_NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
FILE_FLAGS = {"wc_cholinv.hip": ["-fno-slp-vectorize"], "wc_linear.hip": _NO_PACKED_FP32, "wc_gemm_nt.hip": _NO_PACKED_FP32,
              "wc_gemm_codes.hip": _NO_PACKED_FP32, "wc_linear_few.hip": _NO_PACKED_FP32, "wc_experts.hip": _NO_PACKED_FP32}


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    deps.append(os.path.join(os.path.dirname(HERE), "include", "nncf_amd_wc.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=True):
    if not force and not _stale():
        return LIB
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    objs = []
    procs = []
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    for src in sources():
        obj = os.path.join(HERE, "build", os.path.basename(src) + ".o")
        objs.append(obj)
        cmd = [hipcc, *FLAGS, *FILE_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError(f"hipcc failed on {src}")
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", LIB]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
