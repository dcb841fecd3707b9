"""OncePerDevice of csrc/common.cuh, on the CPU with a fake device number: no thread goes on ahead of the call it guards."""
import os
import shutil
import subprocess

import pytest

import test_kernel_source_emulation as E

PROGRAM = r'''
static thread_local int g_device = 0;
static bool g_have_device = true;
#undef cudaGetDevice
#define cudaGetDevice(p) (*(p) = g_device, g_have_device ? cudaSuccess : cudaErrorInvalidDevice)
#include "common.cuh"
#include <chrono>

int main() {
  {  // the second thread gets there while the first is in its call
    amct::OncePerDevice once;
    std::atomic<bool> inside{false}, other_back{false}, set{false};
    bool ahead = false;
    std::thread first([&] {
      once.run([&] {
        inside = true;
        for (int i = 0; i < 2000 && !other_back; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
        set = true;
        return cudaSuccess;
      });
    });
    std::thread second([&] {
      while (!inside) std::this_thread::yield();
      if (!once.run([&] { set = true; return cudaSuccess; })) ahead = true;
      ahead = ahead || !set;                     // back from run(): the call must have been made
      other_back = true;
    });
    first.join();
    second.join();
    if (ahead) return 1;
  }
  amct::OncePerDevice once;
  int calls = 0, fail = 1;
  auto set = [&] { ++calls; return fail ? cudaErrorInvalidValue : cudaSuccess; };
  if (once.run(set) || calls != 1) return 2;     // a failure is reported and the call made again
  fail = 0;
  if (!once.run(set) || calls != 2) return 3;
  if (!once.run(set) || calls != 2) return 4;    // done
  g_device = 1;
  if (!once.run(set) || calls != 3) return 5;    // another device
  g_device = 64;
  if (!once.run(set) || !once.run(set) || calls != 5) return 6;    // numbers beyond the table: every time
  g_device = 0;
  g_have_device = false;
  if (!once.run(set) || calls != 6) return 7;
  return 0;
}
'''


def test_nobody_goes_ahead_of_the_first_call(tmp_path):
    if shutil.which('g++') is None or not os.path.exists(os.path.join(E.CUDA_INCLUDE, 'cuda_fp8.h')):
        pytest.skip('needs g++ and the CUDA headers')
    source, program = tmp_path / 'once.cpp', tmp_path / 'once'
    source.write_text(PROGRAM)
    subprocess.check_call(['g++', '-std=c++17', '-O1', '-w', '-include', os.path.join(E.EMU, 'cuda_emu_routing.h'), '-I', E.CUDA_INCLUDE, '-I', E.CSRC,
                           str(source), '-o', str(program), '-lpthread'])
    assert subprocess.run([str(program)], timeout=60).returncode == 0
