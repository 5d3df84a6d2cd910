"""The C++ front's recurrent-block operators: every wrapper compiles against the header alone, refuses what the C ABI refuses
with its message, and returns where there is nothing to do."""
from __future__ import annotations

import os
import subprocess

from matmulfreellmcpu_b200 import build as B

SOURCE = r"""
#include <cstdio>
#include <string>
#include "mmfree_cuda.hpp"
using namespace mmfree::cuda;

template <class F>
int refused(const char* word, F f) {
  try {
    f();
  } catch (const std::runtime_error& e) {
    if (std::string(e.what()).find(word) != std::string::npos) return 0;
    std::printf("%s: %s\n", word, e.what());
    return 1;
  }
  std::printf("%s: not refused\n", word);
  return 1;
}

int main() {
  mmfree_cuda_conv_args c{};
  mmfree_cuda_ssm_args s{};
  int bad = 0;
  bad += refused("add_rmsnorm_quant", [] { add_rmsnorm_quant(nullptr, nullptr, nullptr, 64, nullptr, 0, nullptr, 1, 64, 1e-6f, MMFREE_T_F32, MMFREE_T_S8); });
  bad += refused("int4_matvec", [] { int4_matvec(nullptr, nullptr, 64, nullptr, nullptr, 32, nullptr, nullptr, 1, 64, 8, 32, 0, MMFREE_T_F32, MMFREE_T_F16, MMFREE_T_F32); });
  bad += refused("causal_conv", [&] { causal_conv(c); });
  bad += refused("causal_conv_step", [&] { causal_conv_step(c); });
  bad += refused("selective_scan", [&] { selective_scan(s); });
  bad += refused("selective_step", [&] { selective_step(s); });
  add_rmsnorm_quant(nullptr, nullptr, nullptr, 64, nullptr, 0, nullptr, 0, 64, 1e-6f, MMFREE_T_F32, MMFREE_T_E4M3, 32);
  int4_matvec(nullptr, nullptr, 64, nullptr, nullptr, 32, nullptr, nullptr, 0, 64, 8, 32, 0, MMFREE_T_F32, MMFREE_T_F16, MMFREE_T_F32);
  return bad;
}
"""


def test_the_wrappers(tmp_path):
    src, exe = tmp_path / "front.cpp", tmp_path / "front"
    src.write_text(SOURCE)
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    r = subprocess.run([cxx, "-std=c++17", "-Wall", "-I" + B.INCLUDE, str(src), "-L" + B.LIBDIR, "-lmmfree_cuda", f"-Wl,-rpath,{B.LIBDIR}",
                        "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
