"""What the library remembers of the occupancy calculator's answers, against a
CUDA runtime played by the test: runtime.cu is compiled with its queries
renamed, and no device is needed."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "reflex_b200", "csrc")
HARNESS = r"""
#include <cuda_runtime.h>
#include <cstdio>

static int answer = 0, queries = 0, device = 0;
static cudaError_t status = cudaSuccess;
static cudaError_t fake_occupancy(int* n, const void*, const cudaLaunchConfig_t*) {
  ++queries;
  *n = answer;
  return status;
}
static cudaError_t fake_device(int* d) {
  *d = device;
  return cudaSuccess;
}
static cudaError_t fake_attribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
#define cudaOccupancyMaxActiveClusters fake_occupancy
#define cudaGetDevice fake_device
#define cudaFuncSetAttribute fake_attribute
#include "runtime.cu"

int main() {
  const void* fn = reinterpret_cast<const void*>(&fake_device);
  auto clusters = [&](cudaError_t s, int a, int threads, int smem, int cluster) {
    status = s, answer = a;
    const int n = rfx::max_active_clusters(fn, threads, smem, cluster);
    printf("clusters %d %d\n", n, queries);
  };
  clusters(cudaErrorMemoryAllocation, 9, 320, 1000, 4);  // a query that fails
  clusters(cudaSuccess, 37, 320, 1000, 4);               // and the same one that does not
  clusters(cudaSuccess, 5, 320, 1000, 4);                // known
  clusters(cudaSuccess, 12, 640, 1000, 4);               // more threads
  clusters(cudaSuccess, 11, 320, 2000, 4);               // more shared memory
  clusters(cudaSuccess, 7, 320, 1000, 8);                // larger clusters
  device = 1;
  clusters(cudaSuccess, 30, 320, 1000, 4);               // another device
  device = 0;
  clusters(cudaSuccess, 5, 320, 1000, 4);                // known
  clusters(cudaSuccess, 0, 320, 3000, 4);                // none fits
  clusters(cudaSuccess, 5, 320, 3000, 4);                // known too
  queries = 0;
  auto fits = [&](cudaError_t s, int a, int cluster) {
    status = s, answer = a;
    const bool f = rfx::cluster_fits(fn, dim3(64), 192, 1000, cluster);
    printf("fits %d %d\n", f ? 1 : 0, queries);
  };
  fits(cudaErrorMemoryAllocation, 9, 16);
  fits(cudaSuccess, 9, 16);
  fits(cudaSuccess, 0, 16);
  fits(cudaSuccess, 0, 8);
  fits(cudaSuccess, 9, 8);
}
"""


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    if not shutil.which("nvcc"):
        pytest.skip("needs nvcc")
    at = tmp_path_factory.mktemp("memo")
    (at / "memo.cu").write_text(HARNESS)
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O0", "-std=c++17", "--expt-relaxed-constexpr",
                    "-I", CSRC, "-I", os.path.join(ROOT, "include"), str(at / "memo.cu"), "-o", str(at / "memo"),
                    "-Xlinker", "--unresolved-symbols=ignore-all"], check=True, capture_output=True)
    out = subprocess.run([str(at / "memo")], check=True, capture_output=True, text=True).stdout
    lines = [line.split() for line in out.splitlines()]
    return lambda what: [(int(n), int(q)) for w, n, q in lines if w == what]


def test_active_clusters_are_remembered_by_what_they_depend_on(said):
    """(answer, queries so far): a failed query answers 0 and is asked again;
    threads, shared memory, cluster size and device are told apart."""
    assert said("clusters") == [(0, 1), (37, 2), (37, 2), (12, 3), (11, 4), (7, 5), (30, 6), (37, 6), (0, 7), (0, 7)]


def test_cluster_fits_is_remembered_once_it_is_known(said):
    assert said("fits") == [(0, 1), (1, 2), (1, 2), (0, 3), (0, 3)]
