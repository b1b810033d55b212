"""The bounded wait of the 8-bit cache's prompt kernel gives up and reports.

No call makes one of that kernel's waits run out, so the wait itself (csrc/common.cuh)
is built into a small kernel that waits on a barrier which nothing completes, for the
2 s that every wait has, beside a second warp that must leave when the first gives up.
"""
import ctypes
import os
import shutil
import subprocess
import time
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CSRC = Path(__file__).resolve().parents[1] / "nano-vllm-cpp26_b200" / "csrc"
SITE = 1 << 16
SOURCE = r"""
#define NVLLM_WHOLE_PROGRAM
#include "common.cuh"
using namespace nvllm;
__global__ void wait_kernel(uint32_t* status, uint32_t* info, uint32_t* left, int complete) {
    __shared__ uint64_t bars[3];
    __shared__ uint32_t abort;
    if (threadIdx.x == 0) {
        mbar_init(&bars[1], 1);
        mbar_init(&bars[2], 1);
        abort = 0;
        fence_barrier_init();
    }
    __syncthreads();
    if (threadIdx.x == 0 && complete) {
        mbar_arrive(&bars[1]);
        mbar_arrive(&bars[2]);
    }
    const int who = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
        if (who == 1 && !complete) {  // starts its own wait a little later
            const uint64_t t0 = global_ns();
            while (global_ns() - t0 < 100000000ull) {}
        }
        left[who] = mbar_wait_or_abort(&bars[1 + who], 0, &abort);
    }
    __syncthreads();
    if (threadIdx.x == 0 && abort != 0) report_abort(status, info, kStatusInKv8Tc, abort, bars);
}
extern "C" int run(uint32_t* status, uint32_t* info, uint32_t* left, int complete) {
    wait_kernel<<<1, 64>>>(status, info, left, complete);
    return cudaDeviceSynchronize();
}
"""


def test_a_wait_that_nothing_ends_gives_up_and_says_where(tmp_path):
    import torch
    nvcc = shutil.which("nvcc") or os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    (tmp_path / "wait.cu").write_text(SOURCE)
    lib = tmp_path / "libwait.so"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++20", "-shared", "-Xcompiler", "-fPIC",
                    f"-I{CSRC}", str(tmp_path / "wait.cu"), "-o", str(lib)], check=True)
    run = ctypes.CDLL(str(lib)).run
    run.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    words = torch.zeros(16, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    at = words.data_ptr()
    assert run(at, at + 16, at + 32, 1) == 0
    assert words.tolist()[:8] == [0] * 8 and words.tolist()[8:10] == [1, 1]
    words.fill_(0)
    torch.cuda.synchronize()
    t0 = time.monotonic()
    assert run(at, at + 16, at + 32, 0) == 0
    waited = time.monotonic() - t0
    got = words.tolist()
    assert 1.9 <= waited < 4.0, waited       # the second warp did not wait its own 2 s out
    assert got[0] == SITE | 2                # the timeout and the kernel's bit
    assert got[4:7] == [SITE | 1, 1, 0]      # its record: the kernel, the barrier's place, the CTA
    assert got[8:10] == [0, 0]               # both left without the phase
