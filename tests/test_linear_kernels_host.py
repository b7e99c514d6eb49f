"""CPU: the sizes that the GPU tests of the 8-bit product run at reach every kernel that the rule knows."""
import os
import shutil
import subprocess

import pytest

from conftest import REPO
from linear_shapes import CASES, SHAPES


def test_the_sizes_of_the_gpu_tests_reach_every_kernel(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src = tmp_path / "rule.cpp"
    src.write_text(r"""
#include "linear_i8.hip.h"
#include <cstdio>
int main()
{
    unsigned m, n, k;
    int whole;
    while (scanf("%u %u %u %d", &m, &n, &k, &whole) == 4) {
        switch (apr::linear_variant(m, n, k, whole, 256)) {
        case apr::kLinear256: puts("kLinear256"); break;
        case apr::kLinear128: puts("kLinear128"); break;
        case apr::kLinear64Deep: puts("kLinear64Deep"); break;
        case apr::kLinear64: puts("kLinear64"); break;
        case apr::kLinearFew: puts("kLinearFew"); break;
        default: return 1;
        }
    }
    return 0;
}
""")
    exe = tmp_path / "rule"
    csrc = os.path.join(REPO, "apr_amd", "csrc")
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-I", csrc, "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, timeout=300)
    sizes = "\n".join(f"{m} {n} {k} {int(whole)}" for _, whole, m, n, k in CASES)
    out = subprocess.run([str(exe)], input=sizes, check=True, capture_output=True, text=True, timeout=60).stdout.split()
    assert out == [kernel for kernel, *_ in CASES]
    # rows at any alignment have two of the five
    assert {k for k, whole in SHAPES if whole} == {"kLinear256", "kLinear128", "kLinear64Deep", "kLinear64", "kLinearFew"}
    assert {k for k, whole in SHAPES if not whole} == {"kLinear128", "kLinearFew"}
