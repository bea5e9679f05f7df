"""The lookup of the driver's tensor map encoder (csrc/tcgen05.cuh) from several threads at once, on the CPU: the
runtime's cudaGetDriverEntryPoint is replaced by one that takes its time."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

SOURCE = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#include "tcgen05.cuh"
static std::atomic<int> calls{0};
extern "C" cudaError_t cudaGetDriverEntryPoint(const char*, void** p, unsigned long long, cudaDriverEntryPointQueryResult* q) {
    calls++;
    std::this_thread::sleep_for(std::chrono::milliseconds(300));
    *p = (void*)0x1000;
    if (q) *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
int main() {
    std::atomic<int> missing{0};
    std::vector<std::thread> all;
    for (int i = 0; i < 8; i++) all.emplace_back([&] { missing += kmc::tensor_map_encode() == nullptr; });
    for (auto& t : all) t.join();
    printf("missing %d calls %d\n", missing.load(), calls.load());
    return 0;
}
"""


def test_every_thread_gets_the_entry_point(tmp_path):
    from mlx_kmeans_b200 import build
    nvcc = shutil.which("nvcc") or build.nvcc()
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "lookup.cu", tmp_path / "lookup"
    src.write_text(SOURCE)
    r = subprocess.run([nvcc, *build.ARCH, "-std=c++17", "-cudart", "shared", "-I", os.path.join(ROOT, "mlx_kmeans_b200", "csrc"),
                        str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "lib64")
    r = subprocess.run([str(exe)], capture_output=True, text=True, env={**os.environ, "LD_LIBRARY_PATH": lib})
    assert r.stdout.split() == ["missing", "0", "calls", "1"], r.stdout + r.stderr
