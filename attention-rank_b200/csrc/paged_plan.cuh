// How the paged attention kernels share out a batch: the units of every sequence form one line, cut
// into equal parts wherever sequences begin or end. Each CTA finds its part from the batch's device
// arrays by itself.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace arb {

struct PlanPlace {
  int sequence;
  int64_t before;  // units before the sequence
};

template <int kCount>  // threads of the block, a multiple of 32
struct PlanScratch {
  int64_t sums[kCount / 32];
  PlanPlace place;
};

#ifdef __CUDACC__

// Inclusive sum over the block's threads, and the block's total.
template <int kCount>
__device__ __forceinline__ int64_t plan_scan(int64_t mine, int64_t& total, PlanScratch<kCount>& scratch) {
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  int64_t sum = mine;
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, sum, offset);
    if (lane >= offset) sum += other;
  }
  if (lane == 31) scratch.sums[warp] = sum;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kCount / 32; ++w) {
    if (w == warp) sum += total;
    total += scratch.sums[w];
  }
  __syncthreads();
  return sum;
}

// Units of the whole batch; units(s) gives a sequence's.
template <int kCount, typename Units>
__device__ __forceinline__ int64_t plan_total(int sequences, PlanScratch<kCount>& scratch, Units units) {
  int64_t mine = 0;
  for (int s = threadIdx.x; s < sequences; s += kCount) mine += units(s);
  int64_t total;
  plan_scan<kCount>(mine, total, scratch);
  return total;
}

// The sequence that holds unit `unit` (below the total).
template <int kCount, typename Units>
__device__ __forceinline__ PlanPlace plan_locate(int sequences, int64_t unit, PlanScratch<kCount>& scratch, Units units) {
  int64_t before = 0;
  for (int base = 0; base < sequences; base += kCount) {
    const int s = base + threadIdx.x;
    const int64_t mine = s < sequences ? units(s) : 0;
    int64_t all;
    const int64_t sum = before + plan_scan<kCount>(mine, all, scratch);
    if (unit >= sum - mine && unit < sum) scratch.place = {s, sum - mine};
    before += all;
    if (unit < before) break;
  }
  __syncthreads();
  return scratch.place;
}

// Parts the line is cut into: one a CTA, each of at least one unit.
__device__ __forceinline__ int plan_parts(int64_t total, int ctas) {
  return static_cast<int>(min(total, static_cast<int64_t>(ctas)));
}
// Where part c of `parts` begins, and the part that holds a unit.
__device__ __forceinline__ int64_t part_begin(int64_t total, int c, int parts) { return total * c / parts; }
__device__ __forceinline__ int part_of(int64_t total, int64_t unit, int parts) {
  return static_cast<int>(((unit + 1) * parts - 1) / total);
}

// Partial sums of a tile that several CTAs share. A CTA has two slots: 1 for a tile that begins in its
// part, 0 for one that began before it.
template <int kRows, int kDim>
struct PartialSums {
  float* sums;    // [2 ctas][kRows][kDim], not divided by the rows' sums
  float2* stats;  // [2 ctas][kRows]: reference and sum
  __device__ __forceinline__ PartialSums(void* workspace, int ctas)
      : sums(static_cast<float*>(workspace)),
        stats(reinterpret_cast<float2*>(sums + static_cast<int64_t>(2) * ctas * kRows * kDim)) {}
};

#endif  // __CUDACC__

constexpr int64_t partial_bytes(int rows, int dim, int ctas) {
  return static_cast<int64_t>(2) * ctas * rows * (dim * sizeof(float) + sizeof(float2));
}

// sum over i < n of floor((a i + b) / m), by Euclid's algorithm on (m, a): whole multiples of m leave
// closed sums, and counting the lattice points below the line that remains by columns instead of rows
// swaps m and a.
__host__ __device__ inline int64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  int64_t sum = 0;
  while (n > 0) {
    const uint32_t a_whole = a / m, b_whole = b / m;
    sum += static_cast<int64_t>(n) * (n - 1) / 2 * a_whole + static_cast<int64_t>(n) * b_whole;
    a -= a_whole * m;
    b -= b_whole * m;
    const uint64_t top = static_cast<uint64_t>(a) * n + b;
    if (top < m) break;
    n = static_cast<uint32_t>(top / m);
    b = static_cast<uint32_t>(top - static_cast<uint64_t>(n) * m);
    const uint32_t swap = m;
    m = a;
    a = swap;
  }
  return sum;
}

// A sequence's new tokens in tiles of `step`: tile t holds tokens [t step, min((t + 1) step, q_len)).
constexpr int kChunkBlock = 128;  // keys a block

struct ChunkTile {
  int first_position;  // of the tile's first token; may be negative
  int last_position;   // of its last token
  int first_key;       // smallest key any row sees (0 when none)
  int block_begin;     // key blocks [block_begin, block_begin + blocks)
  int blocks;          // at least 1
};

__host__ __device__ inline ChunkTile chunk_tile(int q_len, int kv_len, int step, int window, int t) {
  ChunkTile c;
  const int first = kv_len - q_len;
  c.first_position = first + t * step;
  c.last_position = first + (q_len - t * step < step ? q_len : (t + 1) * step) - 1;
  c.first_key = window > 0 && c.first_position >= window ? c.first_position - window + 1 : 0;
  c.block_begin = c.first_key / kChunkBlock;
  const int end = c.last_position < 0 ? 0 : c.last_position / kChunkBlock + 1;
  c.blocks = end - c.block_begin > 1 ? end - c.block_begin : 1;
  return c;
}

// Key blocks of all tiles of a sequence: the sum of chunk_tile(...).blocks in closed form. Without the
// tiles whose every position is negative (one block each), the ends are ceilings and the window's
// beginnings floors of arithmetic sequences over kChunkBlock.
__host__ __device__ inline int64_t chunk_blocks(int q_len, int kv_len, int step, int window) {
  if (q_len <= 0) return 0;
  const uint32_t tiles = (static_cast<uint32_t>(q_len) + step - 1) / step;
  const uint32_t whole = tiles - 1;  // all but the last tile have `step` tokens
  const int first = kv_len - q_len;
  uint32_t empty = 0;  // of the whole tiles, those that end at or before position 0
  if (first < 0) {
    empty = static_cast<uint32_t>(-first) / step;
    empty = empty < whole ? empty : whole;
  }
  const uint32_t end = static_cast<uint32_t>(first + static_cast<int>((empty + 1) * step));  // of the first that is not
  int64_t blocks = empty;
  if (whole > empty) blocks += floor_sum(whole - empty, kChunkBlock, step, end + kChunkBlock - 1);
  blocks += kv_len > 0 ? (kv_len + kChunkBlock - 1) / kChunkBlock : 1;
  if (window > 0 && window < kv_len) {  // else every window begins at position 0
    const int low = first - window + 1;  // where the first tile's window begins, if that is a position
    uint32_t skipped = 0;
    if (low < 0) skipped = (static_cast<uint32_t>(-low) + step - 1) / step;
    if (skipped < tiles) {
      blocks -= floor_sum(tiles - skipped, kChunkBlock, step,
                          static_cast<uint32_t>(low + static_cast<int>(skipped * step)));
    }
  }
  return blocks;
}

}  // namespace arb
