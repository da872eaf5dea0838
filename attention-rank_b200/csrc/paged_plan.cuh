// How the paged attention kernels share out a batch: the units of every sequence form one line, cut
// into equal parts wherever sequences begin or end. Each CTA finds its part from the batch's device
// arrays by itself.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "paged.h"

namespace arb {

#ifdef __CUDACC__

template <int kCount>  // threads of the block, a multiple of 32
struct PlanScratch {
  int64_t sums[kCount / 32];
  int64_t before;  // units before the sequence (or tile) that was found
  PagedSequence seq;
  int index;
};

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
  return sum;
}

// The line's cut into parts, one a CTA, each of at least one unit: the first `longer` parts have one
// unit more than the others.
struct PlanCut {
  int64_t total;
  int parts;
  int longer;
  int64_t length;
  __device__ __forceinline__ int64_t begin(int part) const { return length * part + min(part, longer); }
  __device__ __forceinline__ int part_of(int64_t unit) const {
    const int64_t in_longer = (length + 1) * longer;
    return unit < in_longer ? static_cast<int>(divide(unit, length + 1))
                            : longer + static_cast<int>(divide(unit - in_longer, length));
  }
  // 32-bit where that does: a 64-bit division takes four times as long
  static __device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    if ((a | b) >> 32 == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
  }
};

// What a CTA's part begins with.
struct PlanPlace {
  PlanCut cut;
  int sequence;
  int64_t before;  // units before the sequence
  PagedSequence seq;
};

// Cuts the batch for `ctas` CTAs and finds where part blockIdx.x begins; units(seq) gives a sequence's.
// False: this CTA has no part. The whole block calls it.
template <int kCount, typename Units>
__device__ __forceinline__ bool plan_part(const PagedBatch& b, int* status, int ctas, PlanScratch<kCount>& scratch,
                                          Units units, PlanPlace& place) {
  const int s = threadIdx.x;
  PagedSequence seq = s < b.sequences ? paged_sequence(b, s, status) : PagedSequence{0, 0, 0};
  int64_t mine = units(seq);
  int64_t all;
  int64_t sum = plan_scan<kCount>(mine, all, scratch);
  PlanCut& cut = place.cut;
  cut.total = all;
  for (int base = kCount; base < b.sequences; base += kCount) {  // more sequences than threads
    int64_t more;
    __syncthreads();
    plan_scan<kCount>(base + s < b.sequences ? units(paged_sequence(b, base + s, status)) : 0, more, scratch);
    cut.total += more;
  }
  cut.parts = static_cast<int>(min(cut.total, static_cast<int64_t>(ctas)));
  if (static_cast<int>(blockIdx.x) >= cut.parts) return false;
  cut.length = PlanCut::divide(cut.total, cut.parts);
  cut.longer = static_cast<int>(cut.total - cut.length * cut.parts);
  const int64_t unit = cut.begin(blockIdx.x);
  int64_t before = 0;
  for (int base = 0;; base += kCount) {
    if (unit >= before + sum - mine && unit < before + sum) {
      scratch.index = base + s;
      scratch.before = before + sum - mine;
      scratch.seq = seq;
    }
    before += all;
    if (unit < before || base + kCount >= b.sequences) break;
    const int next = base + kCount + s;
    seq = next < b.sequences ? paged_sequence(b, next, nullptr) : PagedSequence{0, 0, 0};
    mine = units(seq);
    __syncthreads();
    sum = plan_scan<kCount>(mine, all, scratch);
  }
  __syncthreads();
  place.sequence = scratch.index;
  place.before = scratch.before;
  place.seq = scratch.seq;
  return true;
}

// The index i < count whose units hold `unit`, and the units before it; the whole block calls it.
template <int kCount, typename Units>
__device__ __forceinline__ int plan_find(int count, int64_t unit, PlanScratch<kCount>& scratch, Units units,
                                         int64_t& before_it) {
  int64_t before = 0;
  for (int base = 0; base < count; base += kCount) {
    const int i = base + threadIdx.x;
    const int64_t mine = i < count ? units(i) : 0;
    int64_t all;
    __syncthreads();
    const int64_t sum = before + plan_scan<kCount>(mine, all, scratch);
    if (unit >= sum - mine && unit < sum) {
      scratch.index = i;
      scratch.before = sum - mine;
    }
    before += all;
    if (unit < before) break;
  }
  __syncthreads();
  before_it = scratch.before;
  return scratch.index;
}

// What the joining kernel needs about the tile that the beginning of a CTA's part cuts; written by
// every CTA, `last` is below 0 where there is nothing to join (the part begins with a tile, does not
// exist, or another CTA's beginning cuts the tile first).
struct JoinTile {
  int last;  // the part that holds the tile's last unit
  int sequence;
  int tile;
  int kv_head;
  PagedSequence seq;
  int unused;
};

// Partial sums of a tile that several CTAs share, and what to join. A CTA has two slots: 1 for a tile
// that begins in its part, 0 for one that began before it.
template <int kRows, int kDim>
struct PartialSums {
  float* sums;      // [2 ctas][kRows * kDim], not divided by the rows' sums
  float2* stats;    // [2 ctas][kRows]: reference and sum
  JoinTile* tiles;  // [ctas]
  __device__ __forceinline__ PartialSums(void* workspace, int ctas)
      : sums(static_cast<float*>(workspace)),
        stats(reinterpret_cast<float2*>(sums + static_cast<int64_t>(2) * ctas * kRows * kDim)),
        tiles(reinterpret_cast<JoinTile*>(stats + static_cast<int64_t>(2) * ctas * kRows)) {}
};

// One thread of each CTA leaves its JoinTile. `tile_begin` is the unit at which the tile of the part's
// first unit begins.
__device__ __forceinline__ void leave_join_tile(JoinTile* tiles, const PlanPlace* place, int tile, int kv_head,
                                                int64_t tile_begin, int blocks) {
  JoinTile join{};
  join.last = -1;
  const int part = blockIdx.x;
  if (place != nullptr && part > 0 && tile_begin < place->cut.begin(part) && tile_begin >= place->cut.begin(part - 1)) {
    join.last = place->cut.part_of(tile_begin + blocks - 1);
    join.sequence = place->sequence;
    join.tile = tile;
    join.kv_head = kv_head;
    join.seq = place->seq;
  }
  tiles[part] = join;
}

#endif  // __CUDACC__

constexpr int64_t partial_bytes(int rows, int dim, int ctas) {
  return static_cast<int64_t>(ctas) * (2 * rows * (dim * sizeof(float) + sizeof(float2)) + 32);
}

// sum over i < n of floor((a i + b) / m), by Euclid's algorithm on (m, a): whole multiples of m leave
// closed sums, and counting the lattice points below the line that remains by columns instead of rows
// swaps m and a. Everything stays below 2^32: n < 2^25 and, after the first step, a, b < m <= 256.
__host__ __device__ inline int64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  int64_t sum = 0;
  while (n > 0) {
    const uint32_t a_whole = a / m, b_whole = b / m;
    sum += static_cast<int64_t>(n) * (n - 1) / 2 * a_whole + static_cast<int64_t>(n) * b_whole;
    a -= a_whole * m;
    b -= b_whole * m;
    const uint32_t top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top - n * m;
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
