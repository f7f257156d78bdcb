"""The shared-memory limits of kernels (yggdrasil_b200/csrc/ygg_smem.h) under several host threads: the record of a limit
never says more than the kernel's attribute holds. Built with the host compiler against a fake of the two CUDA calls."""
import subprocess
from pathlib import Path

from conftest import ROOT
from yggdrasil_b200 import build

SOURCE = r"""
#include <unistd.h>
#include <cstdio>
#include <thread>
#include "ygg_smem.h"
static std::atomic<int> attribute, calls;
extern "C" cudaError_t cudaGetDevice(int *device) { *device = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int value) {
    attribute = value, calls++;
    if (value == 200) usleep(300000);   // the larger size is set, its caller not yet back
    return value == 7 ? cudaErrorInvalidValue : cudaSuccess;
}
int main() {
    static ygg::SmemLimits limits, other;
    std::thread large([] { ygg::raise_smem_limit(nullptr, 200, limits); });
    usleep(100000);
    std::thread small([] { ygg::raise_smem_limit(nullptr, 100, limits); });
    large.join(), small.join();
    const int after = attribute, first = calls;
    ygg::raise_smem_limit(nullptr, 150, limits);
    const bool again = calls != first;
    const bool refused = ygg::raise_smem_limit(nullptr, 7, other) != cudaSuccess;
    printf("%d %zu %d %d %zu\n", after, limits.set[0].load(), again, refused, other.set[0].load());
}
"""


def test_a_smaller_size_does_not_undo_a_larger_one(tmp_path):
    source, program = tmp_path / "limits.cpp", tmp_path / "limits"
    source.write_text(SOURCE)
    cuda = Path(build.nvcc()).resolve().parents[1] / "include"
    subprocess.run(["g++", "-std=c++17", "-pthread", "-I", str(cuda), "-I", str(ROOT / "yggdrasil_b200" / "csrc"), str(source),
                    "-o", str(program)], check=True)
    out = subprocess.run([str(program)], check=True, capture_output=True, text=True, timeout=60).stdout
    assert out.split() == ["200", "200", "0", "1", "0"]
