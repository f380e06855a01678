"""csrc/per_device.cuh against a runtime made up for the test (no GPU): what the
host keeps for each device and kernel."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG

CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")

# A device's block may have 1000 + device bytes; a kernel (its number as its
# address) has that many bytes of its own.
FAKE = r"""
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>
#include "per_device.cuh"

thread_local int t_device = 0;
std::atomic<int> g_limit[4][8], g_set, g_lowered;
int g_fail = 0;
extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = t_device; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int d) {
    if (a != cudaDevAttrMaxSharedMemoryPerBlockOptin) return cudaErrorInvalidValue;
    *v = 1000 + d;
    return cudaSuccess;
}
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void* k) {
    *a = cudaFuncAttributes{};
    a->sharedSizeBytes = size_t(k);
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void* k, cudaFuncAttribute a, int v) {
    if (g_fail) return cudaErrorInvalidValue;
    if (a != cudaFuncAttributeMaxDynamicSharedMemorySize) return cudaErrorInvalidValue;
    if (g_limit[t_device & 3][size_t(k)].exchange(v) > v) ++g_lowered;
    ++g_set;
    return cudaSuccess;
}
}
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
static const void* kernel(size_t n) { return reinterpret_cast<const void*>(n); }
int main() {
    using namespace moe_b200;
@BODY@
    std::puts("fine");
    return 0;
}
"""

SMEM_LIMIT = r"""
    static SmemLimit a, b;
    g_fail = 1;
    CHECK(a.open(kernel(3)) == cudaErrorInvalidValue);   // a failure is reported and not kept
    g_fail = 0;
    CHECK(a.open(kernel(3)) == cudaSuccess && g_limit[0][3] == 997);
    CHECK(a.open(kernel(3)) == cudaSuccess && g_set == 1);
    CHECK(b.open(kernel(5)) == cudaSuccess && g_limit[0][5] == 995 && g_set == 2);
    t_device = 2;                                        // another device: its own limit
    CHECK(a.open(kernel(3)) == cudaSuccess && g_limit[2][3] == 999 && g_limit[0][3] == 997 && g_set == 3);
    t_device = 100;                                      // more devices than are kept: set in every call
    CHECK(a.open(kernel(3)) == cudaSuccess && a.open(kernel(3)) == cudaSuccess && g_set == 5);
    // threads: never below what a launch that follows may need
    static SmemLimit c;
    std::vector<std::thread> threads;
    std::atomic<int> bad{0};
    for (int i = 0; i < 8; ++i)
        threads.emplace_back([&, i] {
            t_device = i & 1;
            for (int n = 0; n < 1000; ++n)
                if (c.open(kernel(7)) != cudaSuccess || g_limit[i & 1][7] != 993 + (i & 1)) ++bad;
        });
    for (auto& t : threads) t.join();
    CHECK(bad == 0 && g_lowered == 0);
"""

DEVICE_COUNT = r"""
    static DeviceCount count, other;
    int asked = 0;
    auto ask = [&] { ++asked; return 10 + t_device; };
    CHECK(count.get(ask) == 10 && count.get(ask) == 10 && asked == 1);
    t_device = 3;                                        // another device does not get the first one's
    CHECK(count.get(ask) == 13 && count.get(ask) == 13 && asked == 2);
    t_device = 0;
    CHECK(count.get(ask) == 10 && asked == 2 && other.get(ask) == 10 && asked == 3);
    t_device = 100;
    CHECK(count.get(ask) == 110 && count.get(ask) == 110 && asked == 5);
"""


def run(tmp_path, body):
    gxx = shutil.which("g++")
    if gxx is None or not os.path.exists(os.path.join(CUDA, "include", "cuda_runtime_api.h")):
        pytest.skip("needs g++ and the CUDA headers")
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(FAKE.replace("@BODY@", body))
    subprocess.check_call([gxx, "-std=c++17", "-O1", "-pthread", "-I", os.path.join(PKG, "csrc"), "-I", os.path.join(CUDA, "include"),
                           str(src), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "fine", out.stdout


def test_shared_memory_limit_is_set_once_and_never_lowered(tmp_path):
    run(tmp_path, SMEM_LIMIT)


def test_counts_belong_to_their_device(tmp_path):
    run(tmp_path, DEVICE_COUNT)
