"""What is asked of a GPU is asked of each one (the header by itself, with a made-up cudaGetDevice; no GPU needed)."""
import os
import subprocess

MAIN = r"""
#include "per_device.h"
#include <cstdio>
#include <thread>
#include <vector>
static thread_local int current = 0;
static std::atomic<int> asked[80];
extern "C" cudaError_t cudaGetDevice(int* device) { *device = current; return current < 0 ? cudaErrorNoDevice : cudaSuccess; }
extern "C" cudaError_t cudaGetLastError() { return cudaSuccess; }
struct Answer { int of, twice; };
static b200::PerDevice<Answer> answers;
static bool right(int device) {
  current = device;
  const Answer a = answers([] { if (current >= 0) ++asked[current]; return Answer{current, 2 * current}; });
  return a.of == device && a.twice == 2 * device;
}
int main() {
  std::atomic<int> wrong{0};
  std::vector<std::thread> threads;
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&, t] {
      for (int i = 0; i < 4000; ++i) wrong += !right((i + t) % 64);
    });
  for (auto& t : threads) t.join();
  for (int d = 0; d < 64; ++d) wrong += asked[d] != 1;
  for (int d : {64, 79, -1, 64}) wrong += !right(d);
  wrong += asked[64] != 2;
  static std::atomic<uint64_t> told{0};
  int times = 0;
  for (int d : {0, 1, 0, 1, 63, 70, 70}) { current = d; wrong += !b200::once_per_device(told, [&] { ++times; return true; }); }
  wrong += times != 5;
  current = 2;
  wrong += b200::once_per_device(told, [] { return false; }) || !b200::once_per_device(told, [] { return true; });
  printf("%d wrong\n", wrong.load());
  return wrong != 0;
}
"""


def test_each_device_is_asked_once(pkg, tmp_path):
    (tmp_path / "main.cc").write_text(MAIN)
    cuda = os.path.join(os.path.dirname(os.path.dirname(pkg.build.NVCC)), "include")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", pkg.build.CSRC, "-I", cuda, str(tmp_path / "main.cc"), "-o", str(tmp_path / "main"), "-lpthread"], check=True)
    r = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
