"""The once-per-device setup of the paged operators (vvli_b200/csrc/op_common.cuh), compiled for the host."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "op_common.cuh"
#include <cstdio>
#include <thread>
#include <vector>

int main() {
  vvli::SetupOnce once;
  int calls = 0;
  auto fails = [&] { return ++calls, cudaErrorMemoryAllocation; };
  auto works = [&] { return ++calls, cudaSuccess; };
  if (once(fails) != cudaErrorMemoryAllocation || once(fails) != cudaErrorMemoryAllocation || calls != 2) return 1;
  if (once(works) != cudaSuccess || calls != 3) return 2;  // the failures were not kept
  if (once(fails) != cudaSuccess || calls != 3) return 3;  // the success is
  vvli::SetupOnce shared;
  int ran = 0;
  std::vector<std::thread> threads;
  for (int i = 0; i < 8; ++i)
    threads.emplace_back([&] { shared([&] { return ++ran, cudaSuccess; }); });
  for (auto& t : threads) t.join();
  if (ran != 1) return 4;
  std::puts("ok");
  return 0;
}
"""


def test_only_success_is_kept(tmp_path):
    (tmp_path / "setup.cpp").write_text(PROGRAM)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "vvli_b200", "csrc"), "-I",
                    os.path.join(cuda, "include"), "setup.cpp", "-o", "setup"], cwd=tmp_path, check=True)
    assert subprocess.run([str(tmp_path / "setup")], capture_output=True, text=True, timeout=60).stdout == "ok\n"
