"""Build libapr_amd.so (HIP, gfx950) in-tree with hipcc.  No GPU needed to build."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libapr_amd.so")
SOURCES = ["engine.hip", "operators.hip", "model_parse.cpp", "synth.cpp", "ingest.cpp"]
HEADERS = ["conv.hip.h", "frontend.hip.h", "wino.hip.h", "wino4.hip.h", "wino4_fused.hip.h", "wino_fused.hip.h", "wino_fused8.hip.h", "wino_s2.hip.h", "wino_s2_fused.hip.h", "report.hip.h", "resample.hip.h", "conv12_fused.hip.h", "model_parse.h",
           "engine_view.h", "element.hip.h", "logprob.hip.h", "rowquant.hip.h", "linear_i8.hip.h", os.path.join("..", "..", "include", "apr.h")]


# Off in every build: hipcc -O3 forms v_pk_add_f32 / v_pk_mul_f32 / v_pk_fma_f32 from ordinary float code by itself, and some of their
# operand-select forms have given wrong results on this chip.  Packed fp32 issues at half the rate of scalar fp32, so it costs
# nothing: the ten-hour sweep takes 737.4 ms a step against 736.8 with them.  The host pass warns that it does not know the feature.
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc() -> str:
    for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found")


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    files = [os.path.join(CSRC, s) for s in SOURCES + HEADERS] + [os.path.abspath(__file__)]
    return any(os.path.getmtime(f) > t for f in files)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    cmd = [_hipcc(), "-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-shared", "-pthread",
           "-Wall", "-Wno-unused-function", *NO_PACKED_FP32, "-I", os.path.join(HERE, "..", "include"),
           "-o", LIB] + [os.path.join(CSRC, s) for s in SOURCES]
    if verbose:
        cmd.insert(1, "-Rpass-analysis=kernel-resource-usage")
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd, cwd=CSRC)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
