"""The limit of dynamic LDS (csrc/lds_limit.h) is raised for every kernel, also where several have one type, and once for
each device.  Built by the host compiler with stand-ins for the two runtime calls: it runs without a GPU."""

import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "gptq-2d_amd" / "csrc"

RUNTIME = r"""
#pragma once
#include <vector>
static int device = 0, refuse = 0;
static std::vector<const void*> told;
enum { hipFuncAttributeMaxDynamicSharedMemorySize = 8 };
static int hipGetDevice(int* d) { *d = device; return 0; }
static int hipFuncSetAttribute(const void* f, int, int bytes) {
  if (refuse) return 1;
  if (bytes == 163840) told.push_back(f);
  return 0;
}
"""

PROGRAM = r"""
#include <cstdio>
#include "lds_limit.h"
template <int N> static void kernel(int*) {}
int main() {
  refuse = 1;
  int bad = allow_lds<kernel<1>>() != 1;               // an error is passed on, and nothing remembered
  refuse = 0;
  for (int turn = 0; turn < 3; ++turn)
    for (device = 0; device < 2; ++device)
      bad += allow_lds<kernel<1>>() + allow_lds<kernel<2>>();
  int one = 0, two = 0;
  for (const void* f : told) one += f == (const void*)&kernel<1>, two += f == (const void*)&kernel<2>;
  std::printf("%d %d %d\n", bad, one, two);
}
"""


def test_every_kernel_is_told_on_every_device(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ missing")
    source, program = tmp_path / "told.cpp", tmp_path / "told"
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text(RUNTIME)
    source.write_text(PROGRAM)
    built = subprocess.run(["g++", "-std=c++17", f"-I{tmp_path}", f"-I{CSRC}", str(source), "-o", str(program)], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(program)], capture_output=True, text=True)
    assert ran.stdout.split() == ["0", "2", "2"]
