// Attention of new tokens over a paged KV cache (contract in include/attnrank_b200.h). For a row
// (token at position p, query head h):
//   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = scale log2(e) q . k_j,
//   lse = m + log2 sum_j 2^(x_j - m),
// over the visible positions, in one pass with a running reference m and sum.
//
// Few rows a KV head (single tokens, a few drafted ones: at most 48 rows of new tokens x query heads
// of the group): every K and V value is used once to three times per call, so HBM bounds the kernel (64
// single tokens over up to 8K keys, 1.24 GB: 196 to 201 us, 0.94 to 0.96 of the measured copy). K and V arrive
// in 64-key blocks by TMA (192 KB of ring per SM, above the 45 KB that 6.5 TB/s x 1 us of latency
// needs), and the products run on mma.sync m16n8k16 with the group's rows as its 16 rows: the 128 rows
// of a tcgen05 tile would be 7/8 empty.
//
// Work: the batch's (sequence, KV head, key block) units form one line, cut into equal parts, one for
// each CTA of one resident wave (paged_plan.cuh); a part that holds a whole (sequence, KV head) writes
// its rows, the others write fp32 partial sums that the second kernel joins in order. Every CTA finds
// its part from q_offsets and kv_lengths itself, so no plan is made on the host and a captured graph
// follows the lengths it finds.
// Every mbarrier wait is bounded; a warp whose wait gives up records kStatusWaitTimeout and meets the others at
// the barriers of the rest of its part without computing, and the loading warp leaves after its last copies.
// More rows: paged_attention_tc.cu.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "async_copy.cuh"
#include "common.cuh"
#include "device_once.h"
#include "layer_kernels.h"
#include "paged.h"
#include "paged_plan.cuh"

namespace arb {
namespace {

using namespace async;

constexpr int kBlock = 64;          // keys a block
constexpr int kRows = 16;           // rows a tile
constexpr int kCombineThreads = 256;

// One (sequence, KV head, 16 rows) of the line of work.
struct FewTile {
  int first_position;  // of the first new token; negative when fewer are cached than new
  int first_key;       // smallest key any row sees (0 when none)
  int block_begin;     // key blocks [block_begin, block_begin + blocks)
  int blocks;          // at least 1
};

// 16-row tiles of a sequence's rows, new tokens x query heads of a KV head.
__device__ __forceinline__ int few_row_tiles(const PagedAttentionArgs& a, const PagedSequence& seq) {
  return (seq.q_len * (a.query_heads / a.cache.kv_heads) + kRows - 1) / kRows;
}

// Smallest key that the row at `position` sees; the window may be as large as an int gets.
__device__ __forceinline__ int first_visible(int position, int window) {
  return window > 0 && position >= window ? position - window + 1 : 0;
}

__device__ __forceinline__ FewTile few_tile(const PagedSequence& seq, int window) {
  FewTile t;
  t.first_position = seq.kv_len - seq.q_len;
  t.first_key = first_visible(t.first_position, window);
  t.block_begin = t.first_key / kBlock;
  t.blocks = max(1, (seq.kv_len + kBlock - 1) / kBlock - t.block_begin);
  return t;
}

// Units of a sequence; 0 without new tokens, or with more of them than this form takes.
__device__ __forceinline__ int64_t few_units(const PagedAttentionArgs& a, const PagedSequence& seq, int most) {
  if (seq.q_len == 0 || seq.q_len > most) return 0;
  return static_cast<int64_t>(few_tile(seq, a.sliding_window).blocks) * few_row_tiles(a, seq) * a.cache.kv_heads;
}

// Two CTAs an SM, three stages each. A sequence of 17 rows and more is two or three tiles, whose later
// readings of K and V come from L2: one CTA of eight consumer warps for both tiles, with six stages, had too few
// warps to hide its chains behind (28 rows, 16 sequences over up to 4K keys: 28.3 against 33.0 us).
template <int kDim>
struct FewShared {
  static constexpr int kThreads = 5 * 32;
  static constexpr int kCtasPerSm = 2;
  static constexpr int kStages = 3;
  static constexpr uint32_t kBlockBytes = kBlock * kDim * 2;  // of K, or of V
  static constexpr int kPad = 36;                             // floats a merge row of 32 takes
  uint64_t full[kStages];
  uint64_t empty[kStages];
  volatile int abort;
  int poison[2];  // of this segment and the next, in turn
  PlanScratch<kThreads> plan;
  float2 stats[4][kRows];
  alignas(16) float merge[4][kRows][kPad];  // read as float4
  static constexpr size_t bytes() { return 2 * kStages * kBlockBytes + sizeof(FewShared) + 1024; }
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t address, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t address, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address));
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ void consumer_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ bool nonfinite_half(uint32_t bits) {
  constexpr uint32_t kExponent = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u;
  return (bits & kExponent) == kExponent;
}

// Two V values of keys `key` and `key + 1` of a block that not every row sees whole. A probability of
// zero times a NaN or infinity is NaN, so values outside [first, end) (slots nobody wrote, keys no row
// sees) become 0, and so does a value that is not finite, which `poison` reports: the rows that see
// it get it added at the end.
template <typename T>
__device__ __forceinline__ uint32_t clean_pair(uint32_t pair, int key, int first, int end, bool& poison) {
  const bool in0 = key >= first && key < end;
  const bool in1 = key + 1 >= first && key + 1 < end;
  const bool bad0 = nonfinite_half<T>(pair);
  const bool bad1 = nonfinite_half<T>(pair >> 16);
  poison |= (in0 && bad0) || (in1 && bad1);
  return (in0 && !bad0 ? pair & 0xffffu : 0u) | (in1 && !bad1 ? pair & 0xffff0000u : 0u);
}

// Does every row of the sequence see every key of the block that begins at key0?
__device__ __forceinline__ bool whole_block(const PagedSequence& seq, const FewTile& t, int window, int key0) {
  return key0 + kBlock - 1 <= t.first_position && (window == 0 || key0 >= seq.kv_len - window);
}

// Sums of what clean_pair cleared of columns [column, column + 4) at the keys that the row at `position`
// sees: the values that are not finite, in those of the blocks [begin, end) that not every row sees whole.
// That is a few blocks at either end of what the tile sees, however long the cache is, so that no wait
// for this warp runs out meanwhile.
template <typename T, int kDim>
__device__ __forceinline__ float4 nonfinite_sums(const PagedAttentionArgs& a, int s, const PagedSequence& seq,
                                                 const FewTile& t, int begin, int end, int kv_head, int position, int column) {
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int block = t.block_begin + begin; block < t.block_begin + end; ++block) {
    if (whole_block(seq, t, a.sliding_window, block * kBlock)) continue;
    const int first = max(block * kBlock, first_visible(position, a.sliding_window));
    const int last = min(block * kBlock + kBlock - 1, position);
    for (int key = first; key <= last; ++key) {
      const int page = paged_page(a.cache, a.batch, s, key >> a.cache.page_shift, a.status);
      const int64_t row = ((static_cast<int64_t>(page) * a.cache.kv_heads + kv_head) << a.cache.page_shift) +
                          (key & ((1 << a.cache.page_shift) - 1));
      const T* v = static_cast<const T*>(a.cache.v_pages) + row * kDim + column;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float value = static_cast<float>(v[i]);
        if (!isfinite(value)) sum[i] += value;
      }
    }
  }
  return make_float4(sum[0], sum[1], sum[2], sum[3]);
}

template <typename T, int kDim>
__global__ void __launch_bounds__(FewShared<kDim>::kThreads, FewShared<kDim>::kCtasPerSm)
    paged_attention_few_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                               const __grid_constant__ PagedAttentionArgs a, int most) {
  using Shared = FewShared<kDim>;
  constexpr int kThreads = Shared::kThreads;
  constexpr int kStages = Shared::kStages;
  constexpr uint32_t kBlockBytes = Shared::kBlockBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared& sh = *reinterpret_cast<Shared*>(smem + 2 * kStages * kBlockBytes);
  const uint32_t k_smem = smem_u32(smem);
  const uint32_t v_smem = k_smem + kStages * kBlockBytes;
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&sh.full[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), 4);
    }
    sh.abort = 0;
    sh.poison[0] = sh.poison[1] = 0;
    mbar_init_fence();
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }
  wait_for_producer();
  release_dependents();  // the joining kernel waits for this one's completion by itself
  const PartialSums<kRows, kDim> partials(a.workspace, gridDim.x);
  PlanPlace place;  // the barriers inside also cover the set-up above
  const bool has_part = plan_part<kThreads>(
      a.batch, a.status, gridDim.x, sh.plan,
      [&](const PagedSequence& seq) { return few_units(a, seq, most); }, place);
  if (!has_part) {
    if (tid == 0) leave_join_tile(partials.tiles, nullptr, 0, 0, 0, 0);
    return;
  }

  // walk of the part, the same for every role: segments of one (sequence, KV head)
  int s = place.sequence;
  PagedSequence seq = place.seq;
  FewTile tile = few_tile(seq, a.sliding_window);
  const int64_t begin = place.cut.begin(blockIdx.x);
  int row_tiles = few_row_tiles(a, seq);
  const int first_tile = static_cast<int>(PlanCut::divide(begin - place.before, tile.blocks));
  int kv_head = first_tile / row_tiles;
  int row_tile = first_tile - kv_head * row_tiles;
  int block = static_cast<int>(begin - place.before - static_cast<int64_t>(first_tile) * tile.blocks);
  int64_t left = place.cut.begin(blockIdx.x + 1) - begin;
  if (tid == 0) leave_join_tile(partials.tiles, &place, row_tile, kv_head, begin - block, tile.blocks);
  auto next_tile = [&] {
    block = 0;
    if (++row_tile < row_tiles) return;
    row_tile = 0;
    if (++kv_head < a.cache.kv_heads) return;
    kv_head = 0;
    do {  // `left` units remain, so a sequence with new tokens follows
      seq = paged_sequence(a.batch, ++s, nullptr);
    } while (few_units(a, seq, most) == 0 && s + 1 < a.batch.sequences);
    tile = few_tile(seq, a.sliding_window);
    row_tiles = few_row_tiles(a, seq);
  };

  const int page_rows = min(1 << a.cache.page_shift, kBlock);  // rows of one TMA box
  const int boxes = kBlock / page_rows;
  uint32_t turn = 0;  // blocks done so far: stage turn % kStages, phase turn / kStages

  if (warp == 4) {
    // ---------------------------------------------------------------------------------- producer
    bool ok = true;
    while (ok && left > 0) {
      const int count = static_cast<int>(min(left, static_cast<int64_t>(tile.blocks - block)));
      auto page_at = [&](int b) {  // this lane's page of block b, -1 when no row needs it
        const int key = (tile.block_begin + b) * kBlock + lane * page_rows;
        if (lane >= boxes || key >= seq.kv_len || key + page_rows <= tile.first_key) return -1;
        return paged_page(a.cache, a.batch, s, key >> a.cache.page_shift, a.status);
      };
      int page = page_at(block);
      for (int i = 0; i < count; ++i, ++turn) {
        const int following = i + 1 < count ? page_at(block + i + 1) : -1;  // its latency hides behind the wait
        const int stage = turn % kStages;
        const uint32_t round = turn / kStages;
        // the whole warp goes on or stops; a warp that gave up arrives no more, so a stage that is free
        // has landed as well
        const bool free = round == 0 || mbar_wait(smem_u32(&sh.empty[stage]), (round - 1) & 1, &sh.abort);
        if (!__all_sync(0xffffffffu, free && turn < a.self_test_blocks)) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&sh.full[stage]);
        const uint32_t loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_expect_tx(bar, loads * page_rows * kDim * 2 * 2);
        __syncwarp();
        if (page >= 0) {
          const int key = (tile.block_begin + block + i) * kBlock + lane * page_rows;
          const int row = ((page * a.cache.kv_heads + kv_head) << a.cache.page_shift) +
                          (key & ((1 << a.cache.page_shift) - 1));
          const uint32_t to = stage * kBlockBytes + lane * page_rows * kDim * 2;
          tma_load_3d(k_smem + to, &k_map, 0, row, 0, bar);
          tma_load_3d(v_smem + to, &v_map, 0, row, 0, bar);
        }
        page = following;
      }
      left -= count;
      if (left > 0) next_tile();
    }
    if (!ok && turn < a.self_test_blocks && lane == 0) {
      report_status(a.status, kStatusWaitTimeout);
      sh.abort = 1;
    }
    // the loads in flight land before the shared memory is released, even if no consumer waits for them
    for (uint32_t t = turn > kStages ? turn - kStages : 0; t < turn; ++t) {
      mbar_wait(smem_u32(&sh.full[t % kStages]), (t / kStages) & 1, nullptr);
    }
    return;
  }

  // ------------------------------------------------------------------------------------ consumers
  constexpr int kSegmentBarriers = 1 + 2 * (kDim / 32);  // of a segment, in the join of the warps' sums
  const int group = a.query_heads / a.cache.kv_heads;
  const int quarter = warp;  // the warp's 16 keys of a block
  const int g = lane >> 2;
  const int t4 = lane & 3;
  // this lane's addresses inside a block: [page][64-wide half][row][128 bytes], 16-byte chunks XORed
  // with the row's low bits (the TMA's 128-byte swizzle)
  auto row_offset = [&](int key) {
    const int page = key / page_rows;
    const int row = key - page * page_rows;
    return static_cast<uint32_t>(page * page_rows * kDim * 2 + row * 128);
  };
  const int half_bytes = page_rows * 128;
  const uint32_t k_row = row_offset(quarter * 16 + (lane >> 4) * 8 + (lane & 7));
  const int k_chunk = (lane >> 3) & 1;
  const uint32_t v_row = row_offset(quarter * 16 + ((lane >> 3) & 1) * 8 + (lane & 7));
  const int v_chunk = lane >> 4;
  const uint32_t swizzle = lane & 7;  // both rows are 8i + (lane & 7)
  auto chunk_offset = [&](int chunk) {  // 16-byte chunk 0..kDim/8-1 of the lane's row
    return static_cast<uint32_t>((chunk >> 3) * half_bytes + (((chunk & 7) ^ swizzle) << 4));
  };
  bool ok = true;
  int segment = 0;
  while (left > 0) {
    const int count = static_cast<int>(min(left, static_cast<int64_t>(tile.blocks - block)));
    const int rows = seq.q_len * group;
    // Q as MMA operands: the lane holds rows g and g + 8 of its group's 16
    uint32_t q[kDim / 16][4];
    int last_key[2];   // largest key each of the lane's rows sees, below 0: none
    int first_key[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = row_tile * kRows + e * 8 + g;
      const int token = row / group;
      const bool in = row < rows;
      last_key[e] = in ? tile.first_position + token : -1;
      first_key[e] = first_visible(tile.first_position + token, a.sliding_window);
      const T* from = static_cast<const T*>(a.q) + (seq.q_begin + (in ? token : 0)) * a.q_stride +
                      (kv_head * group + (in ? row - token * group : 0)) * kDim + 2 * t4;
#pragma unroll
      for (int k = 0; k < kDim / 16; ++k) {
        q[k][e] = in ? __ldcg(reinterpret_cast<const uint32_t*>(from + 16 * k)) : 0u;
        q[k][2 + e] = in ? __ldcg(reinterpret_cast<const uint32_t*>(from + 16 * k + 8)) : 0u;
      }
    }
    float o[kDim / 8][4];
#pragma unroll
    for (int d = 0; d < kDim / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
    float reference[2] = {-INFINITY, -INFINITY};
    float l[2] = {0.0f, 0.0f};
    bool poison = false;
    // scores of a block; the next block's are computed ahead of this one's softmax, which hides them
    auto scores = [&](uint32_t at_turn, float (&x)[2][4]) {
      const int stage = at_turn % kStages;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.full[stage]), (at_turn / kStages) & 1, &sh.abort))) return false;
      const uint32_t k_at = k_smem + stage * kBlockBytes + k_row;
#pragma unroll
      for (int n = 0; n < 2; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < kDim / 16; ++k) {
        uint32_t b[4];
        ldmatrix_x4(k_at + chunk_offset(2 * k + k_chunk), b);
        mma_16816<T>(x[0], q[k], b[0], b[1]);
        mma_16816<T>(x[1], q[k], b[2], b[3]);
      }
      return true;
    };
    float x[2][4];
    ok = scores(turn, x);
    for (int i = 0; ok && i < count; ++i, ++turn) {
      float following[2][4];
      if (i + 1 < count) ok = scores(turn + 1, following);
      if (!ok) break;
      const int key0 = (tile.block_begin + block + i) * kBlock;
      const int key = key0 + quarter * 16 + 2 * t4;  // of x[0][0]
      // does every row see every key of the block?
      const bool whole = whole_block(seq, tile, a.sliding_window, key0);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[n][c] *= a.scale_log2;
      }
      if (!whole) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int at = key + 8 * n + (c & 1);
            if (at > last_key[c >> 1] || at < first_key[c >> 1]) x[n][c] = -INFINITY;
          }
        }
      }
      // The reference moves only when a score exceeds it by more than its reach (rounded down, so that none
      // passes further); the row's maximum is only looked for then.
      float top[2];
      bool move = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = fmaxf(fmaxf(x[0][2 * e], x[0][2 * e + 1]), fmaxf(x[1][2 * e], x[1][2 * e + 1]));
        move |= top[e] > __fadd_rd(reference[e], kReferenceReach<T>);
      }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
          const float moved = top[e] - kReferenceBelow<T>;
          if (moved > reference[e]) {
            const float factor = reference[e] == -INFINITY ? 0.0f : ex2_ftz(reference[e] - moved);
            reference[e] = moved;
            l[e] *= factor;
#pragma unroll
            for (int d = 0; d < kDim / 8; ++d) {
              o[d][2 * e] *= factor;
              o[d][2 * e + 1] *= factor;
            }
          }
        }
      }
      uint32_t p[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = reference[e] == -INFINITY ? 0.0f : reference[e];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2_ftz(x[n][2 * e] - base);
          const float p1 = ex2_ftz(x[n][2 * e + 1] - base);
          l[e] += p0 + p1;
          p[2 * n + e] = pack2<T>(p0, p1);  // rounded: see kReferenceBelow
        }
      }
      const int stage = turn % kStages;
      const uint32_t v_at = v_smem + stage * kBlockBytes + v_row;
#pragma unroll
      for (int d = 0; d < kDim / 16; ++d) {
        uint32_t b[4];
        ldmatrix_x4_trans(v_at + chunk_offset(2 * d + v_chunk), b);
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            b[r] = clean_pair<T>(b[r], key + 8 * (r & 1), tile.first_key, seq.kv_len, poison);
          }
        }
        mma_16816<T>(o[2 * d], p, b[0], b[1]);
        mma_16816<T>(o[2 * d + 1], p, b[2], b[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.empty[stage]));
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[n][c] = following[n][c];
      }
    }
    if (!ok) break;

    // ---- join the four warps' sums: common reference, then 32 columns at a time through shared memory
    if (__any_sync(0xffffffffu, poison) && lane == 0) sh.poison[segment & 1] = 1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (t4 == 0) sh.stats[quarter][e * 8 + g] = make_float2(reference[e], l[e]);
    }
    consumer_barrier();
    const bool poisoned = sh.poison[segment & 1] != 0;
    // the other flag's readers have passed the last segment's barriers
    if (quarter == 0 && lane == 0) sh.poison[(segment + 1) & 1] = 0;
    const bool begins = block == 0;
    const bool complete = begins && count == tile.blocks;
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (begins ? 1 : 0);
    auto joined = [&](int row) {  // (reference, sum) of one of the 16 rows over the warps
      float2 all = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int w = 0; w < 4; ++w) all.x = fmaxf(all.x, sh.stats[w][row].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 part = sh.stats[w][row];
        all.y += part.y * (part.x == -INFINITY ? 0.0f : ex2_ftz(part.x - all.x));
      }
      return all;
    };
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float factor = reference[e] == -INFINITY ? 0.0f : ex2_ftz(reference[e] - joined(e * 8 + g).x);
#pragma unroll
      for (int d = 0; d < kDim / 8; ++d) {
        o[d][2 * e] *= factor;
        o[d][2 * e + 1] *= factor;
      }
    }
    // this thread's place in a pass: 16 rows x 32 columns, four columns a thread
    const int merge_row = quarter * 4 + (lane >> 3);
    const int row = row_tile * kRows + merge_row;
    const int token = row / group;
    const int head = kv_head * group + row - token * group;
    const float2 all = joined(merge_row);
    const float inverse = all.y != 0.0f ? 1.0f / all.y : 0.0f;
#pragma unroll
    for (int c = 0; c < kDim / 32; ++c) {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          *reinterpret_cast<float2*>(&sh.merge[quarter][e * 8 + g][d * 8 + 2 * t4]) =
              make_float2(o[4 * c + d][2 * e], o[4 * c + d][2 * e + 1]);
        }
      }
      consumer_barrier();
      if (row < rows) {
        const int column = c * 32 + (lane & 7) * 4;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 part = *reinterpret_cast<const float4*>(&sh.merge[w][merge_row][(lane & 7) * 4]);
          sum.x += part.x;
          sum.y += part.y;
          sum.z += part.z;
          sum.w += part.w;
        }
        if (poisoned) {
          const float4 more = nonfinite_sums<T, kDim>(a, s, seq, tile, block, block + count, kv_head,
                                                      tile.first_position + token, column);
          sum.x += more.x;
          sum.y += more.y;
          sum.z += more.z;
          sum.w += more.w;
        }
        if (complete) {
          T* to = static_cast<T*>(a.out) + (seq.q_begin + token) * a.out_stride + head * kDim + column;
          *reinterpret_cast<uint2*>(to) =
              make_uint2(pack2<T>(sum.x * inverse, sum.y * inverse), pack2<T>(sum.z * inverse, sum.w * inverse));
          if (column == 0 && a.lse != nullptr) {
            a.lse[static_cast<int64_t>(seq.q_begin + token) * a.query_heads + head] =
                all.y != 0.0f ? all.x + log2f(all.y) : -INFINITY;
          }
        } else {
          *reinterpret_cast<float4*>(partials.sums + (slot * kRows + merge_row) * kDim + column) = sum;
          if (column == 0) partials.stats[slot * kRows + merge_row] = all;
        }
      }
      consumer_barrier();
    }
    ++segment;
    left -= count;
    if (left > 0) next_tile();
  }
  if (ok) return;
  // A wait gave up: no later one lasts, but the other warps may have got through this one and stand at the
  // barriers of this segment or the next ones, so this warp meets them there.
  if (lane == 0) {
    report_status(a.status, kStatusWaitTimeout);
    sh.abort = 1;
  }
  while (left > 0) {
    for (int i = 0; i < kSegmentBarriers; ++i) consumer_barrier();
    left -= min(left, static_cast<int64_t>(tile.blocks - block));
    if (left > 0) next_tile();
  }
}

// Joins the parts of the tile that the beginning of part blockIdx.x + 1 cuts, in the order of the CTAs.
template <typename T, int kDim>
__global__ void __launch_bounds__(kCombineThreads) paged_attention_few_join_kernel(const PagedAttentionArgs a, int ctas) {
  // every thread waits, so that this grid does not complete before the one whose sums it reads
  wait_for_producer();
  release_dependents();
  const PartialSums<kRows, kDim> partials(a.workspace, ctas);
  const JoinTile join = partials.tiles[blockIdx.x + 1];
  const int last = join.last;
  if (last < 0) return;
  const PagedSequence seq = join.seq;
  const int kv_head = join.kv_head;
  const int c = blockIdx.x;  // the part in which the tile begins
  const int group = a.query_heads / a.cache.kv_heads;
  const int rows = min(kRows, seq.q_len * group - join.tile * kRows);  // of the tile
  constexpr int kBatch = 8;  // parts whose loads are in flight together
  for (int item = blockIdx.y * kCombineThreads + threadIdx.x; item < rows * (kDim / 4);
       item += gridDim.y * kCombineThreads) {
    const int row = item / (kDim / 4);
    const int column = (item - row * (kDim / 4)) * 4;
    float top = -INFINITY;
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int first = c; first <= last; first += kBatch) {
      float2 stats[kBatch];
      float4 piece[kBatch];
      float high = top;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int part = first + i;
        stats[i] = make_float2(-INFINITY, 0.0f);
        piece[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (part <= last) {
          const int64_t at_row = (static_cast<int64_t>(part) * 2 + (part == c ? 1 : 0)) * kRows + row;
          stats[i] = partials.stats[at_row];
          piece[i] = *reinterpret_cast<const float4*>(partials.sums + at_row * kDim + column);
        }
        high = fmaxf(high, stats[i].x);
      }
      const float keep = top == -INFINITY ? 0.0f : ex2_ftz(top - high);
      sum *= keep;
      o.x *= keep;
      o.y *= keep;
      o.z *= keep;
      o.w *= keep;
      top = high;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float factor = stats[i].x == -INFINITY ? 0.0f : ex2_ftz(stats[i].x - top);
        sum += factor * stats[i].y;
        o.x += factor * piece[i].x;
        o.y += factor * piece[i].y;
        o.z += factor * piece[i].z;
        o.w += factor * piece[i].w;
      }
    }
    const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
    const int seq_row = join.tile * kRows + row;
    const int token = seq_row / group;
    const int head = kv_head * group + seq_row - token * group;
    T* to = static_cast<T*>(a.out) + (seq.q_begin + token) * a.out_stride + head * kDim + column;
    *reinterpret_cast<uint2*>(to) =
        make_uint2(pack2<T>(o.x * inverse, o.y * inverse), pack2<T>(o.z * inverse, o.w * inverse));
    if (column == 0 && a.lse != nullptr) {
      a.lse[static_cast<int64_t>(seq.q_begin + token) * a.query_heads + head] =
          sum != 0.0f ? top + log2f(sum) : -INFINITY;
    }
  }
}

// ------------------------------------------------------------------------------------- launches
// [rows of the pool][kDim] as boxes of 64 columns x `rows` rows x (kDim / 64) halves
template <typename T>
bool encode_pages(CUtensorMap* map, const PagedCache& c, void* pages, int rows) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t pool_rows = (static_cast<cuuint64_t>(c.page_count) * c.kv_heads) << c.page_shift;
  const cuuint64_t dims[3] = {64, pool_rows, static_cast<cuuint64_t>(c.head_dim / 64)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.head_dim) * 2, 128};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(rows), static_cast<cuuint32_t>(c.head_dim / 64)};
  const cuuint32_t element_strides[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(map, type, 3, pages, dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int few_ctas() { return sm_count() * FewShared<128>::kCtasPerSm; }

// Takes the sequences of at most `most` new tokens.
template <typename T, int kDim>
cudaError_t launch_few(const PagedAttentionArgs& a, int most, cudaStream_t stream) {
  using Shared = FewShared<kDim>;
  static_assert(Shared::kCtasPerSm * (Shared::bytes() + 1024) <= 228 * 1024, "the CTAs of an SM share its shared memory");
  int device = 0;
  cudaGetDevice(&device);
  static DeviceOnce configured;  // the shared-memory opt-in is a per-device attribute
  const cudaError_t opted = configured.run(device, [] {
    return cudaFuncSetAttribute(paged_attention_few_kernel<T, kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(Shared::bytes()));
  });
  if (opted != cudaSuccess) return opted;
  CUtensorMap k_map, v_map;
  const int rows = std::min(1 << a.cache.page_shift, kBlock);
  if (!encode_pages<T>(&k_map, a.cache, a.cache.k_pages, rows) ||
      !encode_pages<T>(&v_map, a.cache, a.cache.v_pages, rows)) {
    return cudaErrorInvalidValue;
  }
  const int ctas = few_ctas();
  const cudaError_t status = launch_overlapped(paged_attention_few_kernel<T, kDim>, dim3(ctas),
                                               dim3(Shared::kThreads), Shared::bytes(), stream, k_map, v_map, a, most);
  if (status != cudaSuccess || ctas < 2) return status;
  return launch_overlapped(paged_attention_few_join_kernel<T, kDim>, dim3(ctas - 1, kRows / 8),
                           dim3(kCombineThreads), 0, stream, a, ctas);
}

// Which forms a batch takes. A sequence's rows are its new tokens times the query heads of a KV head.
// Sequences of at most kFewRows rows go to the kernel of this file, which reads the cache at HBM's rate
// where a 256-row tile of the chunk kernel would be nearly empty; the others to the chunk kernel. Only
// what the bound on the new tokens allows for is launched, and a batch of one sequence with a larger
// bound takes the chunk kernel alone: the launches it would save cost more than a short chunk there.
// Both forms, this one first, in us a call in a graph (head_dim 128, fp16, the cache partly in L2):
//   heads x KV heads   rows   1 x 4K keys    16 x 512 keys   16 x 4K keys    64 x 1000 keys
//   7 x 4              28     27.0 / 38.0    18.6 / 19.4     44.4 / 41.9     57.5 / 43.5
//                      42     22.7 / 35.8    20.3 / 19.6     59.7 / 41.8     76.2 / 43.5
//                      63     21.4 / 36.7    23.0 / 19.8     68.9 / 42.6     95.3 / 44.0
//   8 x 4              48     20.1 / 32.9    19.8 / 19.3     59.0 / 41.3     75.2 / 44.0
//   4 x 8              28     22.2 / 31.4    22.4 / 22.5     72.4 / 65.9     106.6 / 78.3
//                      48     22.1 / 34.2    27.8 / 22.5     136.0 / 68.2    145.0 / 74.3
//   1 x 16             28     20.7 / 25.0    35.2 / 33.4     175.2 / 121.3   212.1 / 165.5
//                      48     23.6 / 25.4    49.5 / 33.6     261.0 / 132.3   306.3 / 165.9
// The rule looks at rows alone. That is right for one sequence, and for single tokens, where this kernel is at
// HBM's rate; for many sequences of 28 to 48 rows the chunk kernel is the faster one, most where no heads are
// shared and the cache is long.
constexpr int kFewRows = 48;

struct FormChoice {
  int few_tokens = 0;  // new tokens up to which a sequence takes the few-row form; 0: not launched
  bool chunk = false;  // is the chunk form launched?
};

FormChoice choose_forms(const PagedCache& cache, const PagedBatch& batch, int query_heads) {
  const int group = query_heads / cache.kv_heads;
  FormChoice choice;
  choice.chunk = static_cast<int64_t>(batch.max_query) * group > kFewRows;
  if (!choice.chunk || batch.sequences > 1) choice.few_tokens = kFewRows / group;
  return choice;
}

template <typename T, int kDim>
cudaError_t launch_dim(const PagedAttentionArgs& a, cudaStream_t stream) {
  const FormChoice choice = choose_forms(a.cache, a.batch, a.query_heads);
  cudaError_t status = cudaSuccess;
  if (choice.few_tokens > 0) status = launch_few<T, kDim>(a, choice.few_tokens, stream);
  if (status != cudaSuccess || !choice.chunk) return status;
  // the two forms' partial sums share the workspace: each kernel waits for the one before it
  return launch_paged_attention_chunk(a, choice.few_tokens, stream);
}

}  // namespace

int64_t paged_attention_workspace(const PagedCache& cache, const PagedBatch& batch, int query_heads) {
  const FormChoice choice = choose_forms(cache, batch, query_heads);
  int64_t bytes = choice.chunk ? paged_attention_chunk_workspace(cache.head_dim) : 0;
  if (choice.few_tokens > 0) bytes = std::max(bytes, partial_bytes(kRows, cache.head_dim, few_ctas()));
  return bytes;
}

cudaError_t launch_paged_attention(const PagedAttentionArgs& a, cudaStream_t stream) {
  if (a.batch.tokens <= 0 || a.batch.sequences <= 0) return cudaSuccess;
  if (a.cache.dtype == kActFp16) {
    return a.cache.head_dim == 128 ? launch_dim<__half, 128>(a, stream) : launch_dim<__half, 64>(a, stream);
  }
  return a.cache.head_dim == 128 ? launch_dim<__nv_bfloat16, 128>(a, stream)
                                 : launch_dim<__nv_bfloat16, 64>(a, stream);
}

}  // namespace arb
