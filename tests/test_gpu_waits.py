"""The dense FP8 kernels' waits end when what they wait for never comes: a small kernel around the same two functions, whose
barriers nothing (or something) arrives at."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sgl-afd-plugin_b200", "csrc")

SOURCE = r"""
#include "waits.cuh"
using namespace asap;

// warp 0 waits as a folding warp does, warp 1 as the MMA issuer does at its end; `arrive`: which barriers complete
__global__ void waits(int arrive, uint64_t timeout_ns, uint64_t* out) {
  __shared__ uint64_t bar[2];
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar[0], 1);
    mbar_init(&bar[1], 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (threadIdx.x == 32)
    for (int b = 0; b < 2; ++b)
      if (arrive >> b & 1) mbar_arrive(&bar[b]);
  __syncthreads();
  const uint64_t start = globaltimer_ns();
  if (warp == 0) {
    const bool ok = lin::warp_wait(&bar[0], 0, &abort_flag);
    if (lane == 0) out[0] = ok;
  } else {
    lin::drain_mmas(&bar[1], start + timeout_ns, &abort_flag);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    out[1] = abort_flag;
    out[2] = globaltimer_ns() - start;
  }
}

__global__ void tell(uint64_t status, uint64_t word) {
  report(status, word);
  report(status, word + 1);  // the first report stays
}

extern "C" int run_tell(uint64_t status, uint64_t word) {
  tell<<<1, 1>>>(status, word);
  return cudaDeviceSynchronize() == cudaSuccess ? 0 : 2;
}

extern "C" int run(int arrive, uint64_t timeout_ns, uint64_t* host) {
  uint64_t* dev = nullptr;
  if (cudaMalloc(&dev, 24) != cudaSuccess) return 1;
  waits<<<1, 64>>>(arrive, timeout_ns, dev);
  const cudaError_t err = cudaMemcpy(host, dev, 24, cudaMemcpyDeviceToHost);
  cudaFree(dev);
  return err == cudaSuccess ? 0 : 2;
}
"""


@pytest.fixture(scope="module")
def run(cuda_ok, tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("waits")
    src, so = d / "waits.cu", d / "waits.so"
    src.write_text(SOURCE)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "-shared", "-Xcompiler", "-fPIC",
                    "-cudart", "static", "-I", CSRC, "-o", str(so), str(src)], check=True, timeout=300)
    lib = ctypes.CDLL(str(so))

    def call(arrive, timeout_ns):
        out = (ctypes.c_uint64 * 3)()
        assert lib.run(ctypes.c_int(arrive), ctypes.c_uint64(timeout_ns), out) == 0
        return bool(out[0]), bool(out[1]), out[2] / 1e9

    call.lib = lib
    return call


def test_a_report_reaches_the_next_call(run):
    """A kernel's report in the word that the layers give theirs: the next call raises it, once."""
    from asap_b200 import _native as N
    from asap_b200 import linear

    x = torch.randn(4, 256, device="cuda").bfloat16()
    layer = linear.Fp8Linear.from_float(torch.randn(128, 256, device="cuda"))
    want = layer(x)
    linear.check()
    word = 5 | (18 << 32)  # pipeline timeout
    assert run.lib.run_tell(ctypes.c_uint64(layer._w.status), ctypes.c_uint64(word)) == 0
    with pytest.raises(N.AsapError, match="gave up a wait"):
        layer(x)
    assert torch.equal(layer(x), want)
    assert run.lib.run_tell(ctypes.c_uint64(layer._w.status), ctypes.c_uint64(word)) == 0
    with pytest.raises(N.AsapError, match="'seq': 18"):
        linear.check()
    linear.check()


def test_waits_that_are_over(run):
    ok, gave_up, seconds = run(3, 10 ** 9)
    assert ok and not gave_up and seconds < 0.2


def test_mmas_that_never_complete_end_the_folding_warps_too(run):
    ok, gave_up, seconds = run(0, 10 ** 6)
    assert not ok and gave_up and 0.2 <= seconds < 1.0  # at least 0.2 s, for the MMAs in flight
    ok, gave_up, seconds = run(0, 5 * 10 ** 8)
    assert not ok and gave_up and 0.5 <= seconds < 1.5  # no less than the time that was given
    ok, gave_up, _ = run(1, 10 ** 6)  # the folding warp's partial came
    assert ok and gave_up
