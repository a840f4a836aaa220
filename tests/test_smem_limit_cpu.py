"""What a kernel may be launched with (csrc/smem_limit.h) under host threads, compiled here without CUDA."""
import glob
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "infurnace_b200", "csrc")

PROGRAM = r"""
#include "smem_limit.h"
#include <chrono>
#include <cstdio>
#include <thread>
static IfbSmemLimit limit;
static std::atomic<long> attribute{0};
static std::atomic<bool> inside{false}, done{false};
int main() {
  int sets = 0, failed = 0;
  // nothing to set: up to 48 KB, and what is set already
  failed |= limit.raise(3, 48 * 1024, [&]() { ++sets; return 0; }) != 0 || sets != 0;
  failed |= limit.raise(3, 100000, [&]() { ++sets; return 0; }) != 0 || sets != 1;
  failed |= limit.raise(3, 90000, [&]() { ++sets; return 0; }) != 0 || sets != 1;
  failed |= limit.raise(4, 90000, [&]() { ++sets; return 0; }) != 0 || sets != 2;
  // an error is told and not remembered
  failed |= limit.raise(3, 200000, [&]() { return 7; }) != 7;
  failed |= limit.raise(3, 200000, [&]() { ++sets; return 0; }) != 0 || sets != 3;
  if (failed) return 1;
  // one thread is setting 60 KB when another asks for 200 KB; the first goes on once the other is through, or after 0.3 s
  std::thread a([] {
    limit.raise(0, 60 * 1024, [] {
      inside = true;
      for (int i = 0; i < 300 && !done; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
      attribute = 60 * 1024;
      return 0;
    });
  });
  std::thread b([] {
    while (!inside) std::this_thread::yield();
    limit.raise(0, 200 * 1024, [] { attribute = 200 * 1024; return 0; });
    done = true;
  });
  a.join();
  b.join();
  std::printf("%ld\n", attribute.load());
  return attribute.load() == 200 * 1024 ? 0 : 2;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_a_smaller_size_never_comes_behind_a_larger_one(tmp_path):
    source = tmp_path / "limit.cpp"
    source.write_text(PROGRAM)
    program = str(tmp_path / "limit")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", CSRC, "-o", program, str(source)], check=True)
    for _ in range(3):
        run = subprocess.run([program], capture_output=True, text=True, timeout=60)
        assert run.returncode == 0, run.stdout


def test_sizes_that_differ_by_call_are_set_in_one_place():
    """Elsewhere only a constant of the kernel's is set, or nothing."""
    for path in glob.glob(os.path.join(CSRC, "*.c*")):
        with open(path, encoding="utf-8") as f:
            text = f.read()
        if os.path.basename(path) in ("common.cuh", "linear_tcgen05.cu"):      # the macro; sizes of the configuration
            continue
        assert "cudaFuncAttributeMaxDynamicSharedMemorySize" not in text, os.path.basename(path)
