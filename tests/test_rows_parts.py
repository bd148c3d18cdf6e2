"""CPU test of the few-rows attention's part lengths (geoweave_amd/csrc/gw_rows_parts.h, the code that the kernels
compile), up to the largest sizes that the entry points accept: 0x7FFFF000 keys a sequence, fewer than 4,096
row tiles x key heads where the keys are split. The header is compiled with g++ into a program that checks for each
batch that
  * the length is a positive multiple of 256 and the parts of a tile cover its keys, the last one not empty;
  * all parts fit the launch (tiles + want) and those of cut tiles the workspace (2 want);
and that the length cast to 32 bits before it is bounded fails the same check. No GPU work.
"""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "geoweave_amd" / "csrc"

PROGRAM = r"""
#include <stdio.h>
#include <algorithm>
#include <vector>
#include "gw_rows_parts.h"

static int narrow(int64_t total, int want) {
  const int64_t len = (total + want - 1) / want;
  return (int)((std::max(len, (int64_t)gw::kRowsPart) + gw::kRowsPart - 1) / gw::kRowsPart * gw::kRowsPart);
}

// Row tiles of `tiles` each, of sequences of these lengths.
static int check(const std::vector<int>& lens, int tiles, int want, bool bounded) {
  int64_t total = 0;
  for (int lk : lens) total += (int64_t)tiles * lk;
  const int len = bounded ? gw::rows_part_keys(total, want) : narrow(total, want);
  if (len < gw::kRowsPart || len % gw::kRowsPart) return 1;
  int64_t all = 0, cut = 0;
  for (int lk : lens) {
    const int64_t parts = gw::rows_parts(lk, len);
    if (parts < 1 || parts * len < lk || (parts > 1 && (parts - 1) * (int64_t)len >= lk)) return 1;
    all += parts * tiles;
    if (parts > 1) cut += parts * tiles;
  }
  return all > (int64_t)lens.size() * tiles + want || cut >= 2 * (int64_t)want;
}

int main() {
  int bad[2] = {0, 0}, n = 0;
  uint64_t x = 88172645463325252ull;
  auto rnd = [&](uint64_t m) { x ^= x << 13; x ^= x >> 7; x ^= x << 17; return (int64_t)(x % m); };
  for (int b = 0; b < 2; ++b) {
    const std::vector<int> most(4095, (int)gw::kRowsKeysMax), page(4095, 1 << 30), one(1, (int)gw::kRowsKeysMax);
    for (int want : {1024, 512, 128, 1}) {
      bad[b] += check(most, 1, want, b) + check(page, 1, want, b) + check(one, 1, want, b) + check(one, 4095, want, b) +
                check({}, 1, want, b) + check({0}, 1, want, b) + check({1}, 1, want, b);
    }
    for (int i = 0; i < 20000; ++i, ++n) {
      std::vector<int> lens(1 + rnd(60));
      const int top = 1 + (int)rnd(31);
      for (int& l : lens) l = (int)std::min<int64_t>(rnd(1ull << top), gw::kRowsKeysMax);
      bad[b] += check(lens, 1 + (int)rnd(4095 / lens.size()), 1 << rnd(11), b);
    }
  }
  printf("bounded %d narrow %d of %d\n", bad[1], bad[0], n / 2);
  return bad[1] == 0 && bad[0] > 0 ? 0 : 1;
}
"""


def test_part_lengths_stay_in_range(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not found")
    src = tmp_path / "rows_parts.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "rows_parts"
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    print(res.stdout)
    assert res.returncode == 0, res.stdout
