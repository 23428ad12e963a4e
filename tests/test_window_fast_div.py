"""The division by a launch-time block size that the windowed kernels index with: the
multiplier that the host computes, against plain division, at the values next to a border."""
import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PROGRAM = r"""
#include <stdio.h>
#include "window.cuh"

// what the device does with the host's numbers (__umulhi: the high half of the product)
static int64_t quotient(const win::FastDiv &f, int64_t n) {
  return f.d == 1 ? n : (int64_t)(((uint64_t)n * f.m >> 32) >> f.sh);
}

int main() {
  long bad = 0, seen = 0;
  const int64_t top = (int64_t(1) << 31) - 1;
  auto check = [&](int64_t d) {
    const win::FastDiv f = win::fast_div((int)d);
    const uint64_t up = uint64_t(1) << (32 + f.sh);
    bad += f.d != d || (d > 1 && (f.m < up / d || f.m > up / d + 1));
    auto at = [&](int64_t n) {
      if (n < 0 || n > top) return;
      ++seen;
      bad += quotient(f, n) != n / d;
    };
    const int64_t last = top / d;
    for (int64_t i = 0; i <= 64; ++i)
      for (int64_t k : {i, last - i, last / 64 * i, (last / 3) ^ i})
        for (int64_t o = -1; o <= 1; ++o) at(k * d + o);
    at(top);
  };
  for (int64_t d = 1; d <= 5000; ++d) check(d);
  for (int s = 12; s < 31; ++s)
    for (int64_t o = -3; o <= 3; ++o) check((int64_t(1) << s) + o);
  for (int64_t d = 5001; d <= top; d = d * 9 / 8 + 1) check(d);
  for (int64_t o = 0; o < 4; ++o) check(top - o);
  printf("%ld wrong of %ld\n", bad, seen);
  return bad != 0;
}
"""


def test_quotients_next_to_every_border(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not found")
    src, exe = tmp_path / "fast_div.cu", tmp_path / "fast_div"
    src.write_text(PROGRAM)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1",
                    f"-I{ROOT / 'include'}", f"-I{ROOT / 'vllm-apple_b200' / 'csrc'}", str(src),
                    "-o", str(exe)], check=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout.split()[-1]) > 1_000_000
