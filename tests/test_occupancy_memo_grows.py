"""What the library remembers of the occupancy calculator's answers when many shapes
ask: against a CUDA runtime played by the test, as in test_occupancy_memo.py."""
import shutil
import subprocess

import pytest

import test_occupancy_memo as M

MAIN = r"""
int main() {
  const void* fn[2] = {reinterpret_cast<const void*>(&fake_device), reinterpret_cast<const void*>(&fake_attribute)};
  status = cudaSuccess;
  int wrong = 0;
  for (int turn = 0; turn < 3; ++turn)
    for (int f = 0; f < 2; ++f)
      for (device = 0; device < 2; ++device)
        for (int smem = 0; smem < 500; ++smem)
          for (int cluster = 2; cluster <= 8; cluster *= 2) {
            const int right = 1 + smem + 1000 * cluster + 10000 * device + 100000 * f;
            answer = turn == 0 ? right : -1;
            wrong += rfx::max_active_clusters(fn[f], 320, 1024 + 16 * smem, cluster) != right;
          }
  printf("%d %d\n", queries, wrong);
}
"""


@pytest.mark.skipif(not shutil.which("nvcc"), reason="needs nvcc")
def test_many_shapes_are_asked_for_once_each(tmp_path):
    (tmp_path / "memo.cu").write_text(M.HARNESS[:M.HARNESS.index("int main()")] + MAIN)
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O0", "-std=c++17", "--expt-relaxed-constexpr",
                    "-I", M.CSRC, "-I", M.os.path.join(M.ROOT, "include"), str(tmp_path / "memo.cu"), "-o",
                    str(tmp_path / "memo"), "-Xlinker", "--unresolved-symbols=ignore-all"], check=True, capture_output=True)
    out = subprocess.run([str(tmp_path / "memo")], check=True, capture_output=True, text=True).stdout
    assert out.split() == [str(2 * 2 * 500 * 3), "0"]
