"""The raising of a kernel's shared-memory limit (SmemLimit), on the host with a stand-in for the CUDA
calls: two threads that raise one kernel at once leave a limit that both can launch with."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "vdxs_internal.h"

#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>

static std::mutex mu;
static std::condition_variable cv;
static int limit = 48 * 1024, calls = 0;  // CUDA's side: the last value set stands
static bool other_done = false;

extern "C" cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
    std::unique_lock<std::mutex> lock(mu);
    limit = bytes;
    const bool first = calls++ == 0;
    cv.notify_all();
    // The first caller is held up behind its call until the other thread is through (or waits for it).
    if (first) cv.wait_for(lock, std::chrono::milliseconds(500), [] { return other_done; });
    return cudaSuccess;
}

static void kernel() {}
static vdxs::SmemLimit tracked;
static bool launch(int bytes) {
    return tracked.raise(&kernel, (size_t)bytes) == cudaSuccess && bytes <= limit;
}

int main() {
    const int more = 110 * 1024, less = 60 * 1024;
    std::thread a([=] { tracked.raise(&kernel, more); });
    {
        std::unique_lock<std::mutex> lock(mu);
        cv.wait(lock, [] { return calls > 0; });
    }
    tracked.raise(&kernel, less);
    {
        std::lock_guard<std::mutex> lock(mu);
        other_done = true;
        cv.notify_all();
    }
    a.join();
    for (int bytes : {less, 80 * 1024, more, 50 * 1024, 120 * 1024, less, 40 * 1024})
        if (!launch(bytes)) { std::printf("%d bytes do not launch with a limit of %d\n", bytes, limit); return 1; }
    return 0;
}
"""


def test_two_threads_raise_one_kernel(tmp_path):
    include = next((d for d in ("/usr/local/cuda/include", os.path.join(os.environ.get("CUDA_HOME", ""), "include"))
                    if os.path.exists(os.path.join(d, "cuda_runtime.h"))), None)
    gxx = shutil.which("g++")
    if not include or not gxx:
        pytest.skip("no g++ or CUDA headers")
    src, exe = tmp_path / "limit.cpp", tmp_path / "limit"
    src.write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-pthread", "-I", include, "-I", os.path.join(ROOT, "vindexllm_b200", "csrc"),
                    str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout
