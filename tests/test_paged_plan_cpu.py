"""The closed forms by which the paged attention kernels share out a batch (csrc/paged_plan.cuh), compiled
for the host: tiles against their rows, and the key blocks of a sequence against the sum over its tiles."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "attention-rank_b200" / "csrc"
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include "paged_plan.cuh"
#include <cstdio>
#include <random>
using namespace arb;
static long bad = 0;
static void check(int q, int kv, int step, int window, bool rows) {
  int64_t sum = 0;
  for (int64_t at = 0; at < q; at += step) {
    const int t = static_cast<int>(at / step);
    const ChunkTile c = chunk_tile(q, kv, step, window, t);
    sum += c.blocks;
    if (c.blocks < 1) ++bad;
    if (!rows) continue;
    int64_t low = -1, high = -1;  // keys that any row of the tile sees
    for (int64_t i = at; i < q && i < at + step; ++i) {
      const int64_t p = static_cast<int64_t>(kv) - q + i;
      if (p < 0) continue;
      const int64_t first = window > 0 && p >= window ? p - window + 1 : 0;
      if (low < 0 || first < low) low = first;
      high = p;
    }
    if (high < 0) continue;
    const int64_t begin = static_cast<int64_t>(c.block_begin) * kChunkBlock;
    if (low < c.first_key || low < begin || low >= begin + kChunkBlock) ++bad;
    if (high != c.last_position || high / kChunkBlock + 1 != c.block_begin + static_cast<int64_t>(c.blocks)) ++bad;
  }
  if (chunk_blocks(q, kv, step, window) != sum) {
    if (++bad < 5) std::printf("q %d kv %d step %d window %d\n", q, kv, step, window);
  }
}
int main() {
  std::mt19937 rng(7);
  auto below = [&](int n) { return static_cast<int>(rng() % static_cast<unsigned>(n)); };
  const int largest = 2147483647;
  for (int i = 0; i < 150000; ++i) {
    const int step = 2 * (128 / (1 + below(128)));
    const int q = below(5) == 0 ? below(5) : 1 + below(3000);
    const int kv = below(4) == 0 ? below(4000) : q + below(20000);
    check(q, below(50) == 0 ? 0 : kv, step, below(2) ? 0 : below(10) == 0 ? largest : 1 + below(5000), true);
  }
  for (int i = 0; i < 3000; ++i) {  // to the ends of the ranges
    const int step = 2 * (128 / (1 + below(128)));
    const int q = 1 + below(1 << (1 + below(20)));
    const int kv = largest - 1024 - below(1 << (1 + below(30)));
    check(q, kv, step, below(3) == 0 ? 0 : below(2) ? largest - below(1000) : 1 + below(largest), false);
  }
  check(1 << 24, largest - 1024, 256, 0, false);
  check(1 << 24, 5, 2, 0, false);
  check(1 << 24, (1 << 24) + 100, 18, 4096, false);
  std::printf("bad %ld\n", bad);
  return bad != 0;
}
"""


def test_block_counts_are_the_sums_over_tiles(tmp_path):
    if not Path(NVCC).exists():
        pytest.skip("no nvcc")
    source, program = tmp_path / "plan.cu", tmp_path / "plan"
    source.write_text(PROGRAM)
    built = subprocess.run([NVCC, "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr",
                            f"-I{CSRC}", str(source), "-o", str(program)], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stdout
