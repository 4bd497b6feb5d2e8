"""The helper that sets a kernel's shared memory once (csrc/smem_attr.h), against a fake of the CUDA call: first calls of
several sizes from threads of their own. CPU only."""

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PROGRAM = r"""
#include <unistd.h>

#include <cstdio>
#include <thread>

#include "smem_attr.h"

static std::atomic<int> limit{0}, calls{0};
extern "C" cudaError_t cudaGetDevice(int* device) { *device = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
  ++calls;
  if (bytes == 100) usleep(300000);                       // the smaller size's call takes its time
  limit = bytes;
  return cudaSuccess;
}

int main() {
  static std::atomic<int> done[trnopt::kMaxDevices];
  const void* fn = reinterpret_cast<const void*>(main);
  std::thread small([&] { trnopt::smem_attr_once(fn, 100, done); });
  usleep(100000);
  std::thread large([&] { trnopt::smem_attr_once(fn, 200, done); });
  small.join();
  large.join();
  trnopt::smem_attr_once(fn, 200, done);
  const int before = calls;
  trnopt::smem_attr_once(fn, 150, done);                  // covered: no call
  std::printf("%d %d\n", (int)limit, calls - before);
}
"""


def test_a_smaller_size_set_late_does_not_stay(tmp_path):
    cxx = shutil.which("g++")
    include = next((p for p in map(Path, ("/usr/local/cuda/include",)) if (p / "cuda_runtime.h").exists()), None)
    if cxx is None or include is None:
        pytest.skip("no C++ compiler or CUDA headers")
    (tmp_path / "main.cpp").write_text(PROGRAM)
    exe = tmp_path / "main"
    subprocess.run([cxx, "-std=c++17", "-pthread", f"-I{include}", f"-I{ROOT / 'trainium-sinkhorn_b200' / 'csrc'}",
                    str(tmp_path / "main.cpp"), "-o", str(exe)], check=True, timeout=120)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split() == ["200", "0"]
