"""Host-side launch helpers of csrc/kernels against a fake CUDA runtime (no GPU)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAKE = r"""
#include <cuda_runtime_api.h>
#include <map>
#include <utility>
int device = 0, sets = 0;
std::map<std::pair<const void*, int>, int> limits;
extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int d) {
  *v = a == cudaDevAttrMaxSharedMemoryPerBlockOptin ? 232448 + 1024 * d : a == cudaDevAttrMultiProcessorCount ? 100 + d : 0;
  return cudaSuccess;
}
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) { a->sharedSizeBytes = 448; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute, int v) {
  sets++, limits[{f, device}] = v;
  return cudaSuccess;
}
// what the compiler's registration of the (empty) device code calls
void** __cudaRegisterFatBinary(void*) { static void* h; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
char __cudaInitModule(void**) { return 0; }
}
"""
PROGRAM = r"""
#include "common.cuh"
#include <cstdio>
#include <map>
extern int device, sets;
extern std::map<std::pair<const void*, int>, int> limits;
int main() {
  static int a, b;
  for (device = 0; device < 3; device++)
    for (int again = 0; again < 2; again++)
      for (const void* k : {(const void*)&a, (const void*)&b}) moet_allow_max_smem(k);
  for (device = 0; device < 3; device++)
    for (const void* k : {(const void*)&a, (const void*)&b})
      if (limits[{k, device}] != 232448 + 1024 * device - 448) {
        printf("device %d: %d\n", device, limits[{k, device}]);
        return 1;
      }
  printf("%d\n", sets);
  return sets == 6 ? 0 : 2;
}
"""


SM_PROGRAM = r"""
#include "kv4.cuh"
#include <cstdio>
extern int device;
int main() {
  for (device = 0; device < 3; device++) {
    printf("%d\n", moet::kv4::sm_count());
    if (moet::kv4::sm_count() != 100 + device) return 1;
  }
  return 0;
}
"""


def build_and_run(tmp_path, program):
    src, fake, exe = tmp_path / "program.cu", tmp_path / "fake.cpp", tmp_path / "program"
    src.write_text(program)
    fake.write_text(FAKE)
    subprocess.run(["nvcc", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "none",
                    "-I", os.path.join(ROOT, "csrc", "kernels"), str(src), str(fake), "-o", str(exe)], check=True, timeout=300)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)


needs_nvcc = pytest.mark.skipif(shutil.which("nvcc") is None, reason="no nvcc")


@needs_nvcc
def test_shared_memory_is_allowed_once_per_kernel_and_device(tmp_path):
    """The attribute belongs to a device's context: a second device of one process needs it too."""
    got = build_and_run(tmp_path, PROGRAM)
    assert got.returncode == 0, got.stdout


@needs_nvcc
def test_sm_count_is_the_current_device_s(tmp_path):
    got = build_and_run(tmp_path, SM_PROGRAM)
    assert got.returncode == 0, got.stdout
