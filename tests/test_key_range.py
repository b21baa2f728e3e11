"""The bins in which top_logits looks for the k-th largest key (csrc/key_range.h), with a loop in the place of a block: all of
the k largest keys stay, and few others."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "multimodal_training_b200" / "csrc"

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <cstring>
#include <functional>
#include <vector>
#include "key_range.h"

typedef unsigned long long u64;

// Order-preserving bits of a logit, as in csrc/vocab_rows.cuh for numbers.
unsigned order32(float x) {
  unsigned b;
  memcpy(&b, &x, 4);
  if (b == 0x80000000u) b = 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Rows of: type (0: bf16, 1: fp32), number of logits, logits as fp32 bits with columns, number of questions, and each
// question's k and bound (16 bits that k keys reach).
int main() {
  int f32, k, n, questions;
  unsigned bound;
  while (scanf("%d %d", &f32, &n) == 2) {
    std::vector<u64> list(n);
    for (u64& key : list) {
      unsigned bits, column;
      if (scanf("%u %u", &bits, &column) != 2) return 1;
      float x;
      memcpy(&x, &bits, 4);
      key = (u64)(f32 ? order32(x) : order32(x) >> 16) << 32 | (0xffffffffu - column);
    }
    std::vector<u64> best = list;
    std::sort(best.begin(), best.end(), std::greater<u64>());
    if (scanf("%d", &questions) != 1) return 1;
    while (questions-- > 0) {
      if (scanf("%d %u", &k, &bound) != 2) return 1;
      const int shift = f32 ? 48 : 32;
      unsigned most = 0;
      for (u64 key : list) most = std::max(most, (unsigned)(key >> shift) & 0xffffu);
      KeyRange range(bound, most, shift);
      int need = k, sure = 0, levels = 0, outside = 0;
      for (;;) {
        ++levels;
        int hist[KeyRange::kBins] = {};
        for (u64 key : list)
          if (range.holds(key)) {
            if (range.bin(key) < 0 || range.bin(key) >= KeyRange::kBins) ++outside;
            else ++hist[range.bin(key)];
          }
        int d = KeyRange::kBins - 1, above = 0;
        while (d > 0 && above + hist[d] < need) above += hist[d--];
        range.raise(d);
        sure += above;
        need -= above;
        if (sure + hist[d] <= k + 64 || !range.narrow()) break;
      }
      int left = 0;
      for (u64 key : list) left += key >= range.low;
      printf("%d %d %d %d\n", left, (int)(best[k - 1] >= range.low), levels, outside);
    }
  }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("key_range")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-I", str(CSRC), str(d / "main.cpp"), "-o", str(d / "main")], check=True)
    return d / "main"


def _rows():
    """(name, logits in the order of their columns)"""
    import numpy as np
    rng = np.random.default_rng(0)
    rows = [(f"all {v}", np.full(2048, v)) for v in (-1.0, -0.5, 0.0, 1.0, 2.0, -1e30)]
    for some in (20, 40, 100, 300):
        masked = np.full(2048, -np.inf)
        masked[rng.choice(2048, some, replace=False)] = rng.uniform(-6.0, -0.3, some)
        rows.append((f"{some} log-probabilities", masked))
        sparse = np.zeros(2048)
        sparse[2048 - some:] = rng.uniform(2.0, 40.0, some)
        rows.append((f"{some} late positive logits", sparse))
    rows.append(("normal", rng.normal(size=2048) * 3))
    rows.append(("few values", rng.integers(-2, 3, 2048).astype(float)))
    for e in range(1, 17):                          # a second value at each distance from the first
        two = np.full(2048, -1.0)
        two[1::2] = -2.0 ** e if e < 8 else -1.0 - 2.0 ** (7 - e)
        rows.append((f"two values, {e}", two))
    return rows


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("first_column", [0, 100, 12345])
def test_the_k_largest_keys_stay(program, f32, first_column):
    import numpy as np
    lines, names = [], []
    for name, row in _rows():
        bits = row.astype(np.float32).view(np.uint32)
        if not f32:
            bits = bits & np.uint32(0xffff0000)
        body = " ".join(f"{b} {c}" for c, b in enumerate(bits.tolist(), first_column))
        order = np.where(bits == 0x80000000, 0, bits)
        order = np.sort(np.where(order >> 31 == 1, ~order, order | np.uint32(0x80000000)) >> 16)[::-1]
        asked = []
        for k in [1, 40, 64, 65, *range(72, 256, 20), 256]:
            for bound in sorted({0, int(order[k - 1])}):
                asked.append(f"{k} {bound}")
                names.append((name, k, bound))
        lines.append(f"{f32} {len(row)} {body} {len(asked)} {' '.join(asked)}")
    out = subprocess.run([str(program)], input="\n".join(lines), capture_output=True, text=True, check=True).stdout.split("\n")
    for (name, k, bound), line in zip(names, out):
        left, kth, levels, outside = (int(v) for v in line.split())
        assert k <= left <= k + 64 and kth and not outside, (name, k, bound, left)
        # the first bins have at most 2^8 times the 2^shift keys that 16 bits leave open, further ones a 2^8th each
        assert levels <= (8 if f32 else 6)
