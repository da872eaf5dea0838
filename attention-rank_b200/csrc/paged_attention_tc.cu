// Attention of chunks of new tokens over a paged KV cache on tcgen05 / TMEM (contract in
// include/attnrank_b200.h, formulas in paged_attention.cu).
//
// Rows: the query heads of a KV head are stacked, row = token * group + head, so that they share each
// K and V tile and the causal edge of a tile stays a few tokens wide. A tile is two M = 128 halves of
// floor(128 / group) tokens each; K and V come in 128-key blocks, one or more pages each, by TMA.
// One persistent CTA an SM, 320 threads:
//   warps 0-3, 4-7  softmax of half 0 / 1: thread r owns row r (TMEM lane r) of its half
//   warp 8          TMA: Q of both halves, K and V blocks into a ring of four stages
//   warp 9          tcgen05.mma of both halves
// TMEM: S0 | S1 | O0 | O1, 128 columns each; P (16-bit) overwrites its S. Per half and block:
//   S = Q K^T;  softmax warps read S and write P, 96 keys, then 32;  O += P V starts with the first
//   while the others are being computed;  the next S follows behind it.
// While one half's products run, the other half's softmax does.
// Bounds: the products of a block take the tensor pipe 2048 clocks, its 2 x 128 x 128 exponentials the
// SFU as many (16 a clock and SM). A half's chain, scores - softmax - P V - next scores, is about 3400
// clocks long, of which the pipe works 2048; two 4K chunks over up to 8K keys (825 GFLOP) take 780 to
// 860 us, 0.59 to 0.64 of the measured burst, at clocks that fall to 1.55 GHz under the power limit.
//
// Work: the (tile, KV head, key block) units form one line that is cut into equal parts, one a CTA
// (paged_plan.cuh); tiles that a part does not hold whole leave fp32 partial sums, which the joining
// kernel adds up in order.
// Masked rows and positions: scores by selection; V values that not every row may see, by clearing the
// tile's copy (slots past the end, values that are not finite) before the product.
// Every mbarrier wait is bounded; on expiry the kernel records kStatusWaitTimeout, loads no more, runs
// through the rest without waiting, waits (bounded) for its own MMAs and copies, frees TMEM and returns.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "async_copy.cuh"
#include "common.cuh"
#include "device_once.h"
#include "layer_kernels.h"
#include "paged.h"
#include "paged_plan.cuh"
#include "tensor_core.cuh"

namespace arb {
namespace {

using namespace async;
using namespace tc;

constexpr int kRows = 128;                          // rows of a half tile
constexpr int kThreads = 320;
constexpr int kStages = 4;
constexpr uint32_t kHalfBytes = 128 * 128;          // 128 rows of 64 16-bit values
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kTmemO = 256;
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 32;                       // rows of a tile that one joining CTA takes
constexpr int kChains = 4;                          // independent accumulators per row reduction

struct __align__(16) Control {
  uint64_t q_full;
  uint64_t q_empty;
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t s_full[2];
  uint64_t p_full[2][2];
  uint64_t o_full[2];
  uint64_t o_free[2];
  uint64_t clean[2];
  uint64_t done;
  uint32_t tmem_base;
  volatile int abort;
  unsigned poison;  // bit segment % 32: V held a value that is not finite where some row may not look
  PlanScratch<kThreads> plan;
};

template <int kDim>
struct Layout {
  static constexpr uint32_t kOperand = kHalfBytes * (kDim / 64);  // 128 rows of K, V, or half a tile's Q
  static constexpr uint32_t kRing = 2 * kOperand;
  static constexpr uint32_t kControl = kRing + kStages * kOperand;
  static constexpr size_t bytes() { return kControl + sizeof(Control) + 1024; }
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

struct ChunkArgs {
  PagedAttentionArgs a;
  int half_tokens;  // tokens of half a tile
  int few;          // sequences of at most so many new tokens are left out
  uint32_t idesc_s;
  uint32_t idesc_o;
};

// Units of a sequence: the key blocks of all its tiles, for every KV head.
__device__ __forceinline__ int64_t chunk_units(const ChunkArgs& c, const PagedSequence& seq) {
  if (seq.q_len <= c.few) return 0;
  return chunk_blocks(seq.q_len, seq.kv_len, 2 * c.half_tokens, c.a.sliding_window) * c.a.cache.kv_heads;
}

// One segment: the part of a (tile, KV head) that one CTA does.
struct Walk {
  PagedSequence seq;
  ChunkTile tile;
  int s, t, kv_head;
  int block;     // first block of the segment, relative to the tile's
  int count;     // its blocks
  int64_t left;  // units of the part from this segment on
  // blocks of the segment [begin, end) that any row of a half sees, relative to the tile's
  __device__ __forceinline__ void half_range(int half, int half_tokens, int window, int& begin, int& end) const {
    const int first = tile.first_position + half * half_tokens;
    const int last = min(first + half_tokens - 1, tile.last_position);
    begin = end = block;
    if (first > tile.last_position || last < 0) return;
    const int first_key = window > 0 && first >= window ? first - window + 1 : 0;
    begin = max(block, first_key / kChunkBlock - tile.block_begin);
    end = max(begin, min(block + count, last / kChunkBlock + 1 - tile.block_begin));
  }
  // does every row of the tile see every key of block b?
  __device__ __forceinline__ bool whole(int b, int window) const {
    const int key = (tile.block_begin + b) * kChunkBlock;
    return key + kChunkBlock - 1 <= tile.first_position && (window == 0 || key > tile.last_position - window);
  }
};

__device__ __forceinline__ void walk_tile(Walk& w, const ChunkArgs& c) {
  w.tile = chunk_tile(w.seq.q_len, w.seq.kv_len, 2 * c.half_tokens, c.a.sliding_window, w.t);
  w.count = static_cast<int>(min(w.left, static_cast<int64_t>(w.tile.blocks - w.block)));
}
__device__ __forceinline__ bool walk_next(Walk& w, const ChunkArgs& c) {
  w.left -= w.count;
  if (w.left <= 0) return false;
  w.block = 0;
  if (++w.kv_head == c.a.cache.kv_heads) {
    w.kv_head = 0;
    if (++w.t * 2 * c.half_tokens >= w.seq.q_len) {
      w.t = 0;
      do {  // units remain, so a sequence of this form follows
        w.seq = paged_sequence(c.a.batch, ++w.s, nullptr);
      } while (w.seq.q_len <= c.few && w.s + 1 < c.a.batch.sequences);
    }
  }
  walk_tile(w, c);
  return true;
}

// Of a pair of 16-bit values, the sign bits of those that are not finite (exponent all ones: adding
// one to it carries into the sign's place).
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_pair(uint32_t pair) {
  constexpr uint32_t kExponents = std::is_same_v<T, __half> ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t kOnes = std::is_same_v<T, __half> ? 0x04000400u : 0x00800080u;
  return ((pair & kExponents) + kOnes) & 0x80008000u;
}
// The pair with its values that are not finite cleared.
template <typename T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t pair) {
  return pair & ~((nonfinite_pair<T>(pair) >> 15) * 0xffffu);
}

// Adds to a row, written by this thread, what was cleared of the segment's V at the keys [row_first,
// row_last] it sees: the values that are not finite, in the blocks that not every row of the tile sees
// whole. That is a few blocks at either end of what the tile sees, however long the cache is, so that no
// wait for this warp runs out meanwhile. `out` is the row in the 16-bit result, or NULL and `sums` its
// place in the partial sums.
template <typename T, int kDim>
__device__ __noinline__ void add_nonfinite(const PagedAttentionArgs& a, const Walk w, int row_first, int row_last, T* out,
                                           float* sums) {
  for (int b = w.block; b < w.block + w.count; ++b) {
    if (w.whole(b, a.sliding_window)) continue;
    const int key0 = (w.tile.block_begin + b) * kChunkBlock;
    for (int key = max(key0, row_first); key <= min(key0 + kChunkBlock - 1, row_last); ++key) {
      const int page = paged_page(a.cache, a.batch, w.s, key >> a.cache.page_shift, a.status);
      const int64_t row = ((static_cast<int64_t>(page) * a.cache.kv_heads + w.kv_head) << a.cache.page_shift) +
                          (key & ((1 << a.cache.page_shift) - 1));
      const uint4* v = reinterpret_cast<const uint4*>(static_cast<const T*>(a.cache.v_pages) + row * kDim);
#pragma unroll 4
      for (int i = 0; i < kDim / 8; ++i) {
        const uint4 raw = v[i];
        if ((nonfinite_pair<T>(raw.x) | nonfinite_pair<T>(raw.y) | nonfinite_pair<T>(raw.z) | nonfinite_pair<T>(raw.w)) == 0) {
          continue;
        }
        float value[8];
        unpack8<T>(raw, value);
        for (int j = 0; j < 8; ++j) {
          const int column = 8 * i + j;
          if (isfinite(value[j])) continue;
          if (out != nullptr) {
            out[column] = static_cast<T>(static_cast<float>(out[column]) + value[j]);
          } else {
            sums[(column >> 2) * (2 * kRows * 4) + (column & 3)] += value[j];
          }
        }
      }
    }
  }
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attention_chunk_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ ChunkArgs c) {
  constexpr uint32_t kOperand = Layout<kDim>::kOperand;
  constexpr int kHalves = kDim / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Control& ctl = *reinterpret_cast<Control*>(smem + Layout<kDim>::kControl);
  const uint32_t q_smem = smem_u32(smem);
  const uint32_t ring = q_smem + Layout<kDim>::kRing;
  const PagedAttentionArgs& a = c.a;
  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be the same in the whole warp
  const int lane = tid & 31;
  const int window = a.sliding_window;

  if (tid == 0) {
    mbar_init(smem_u32(&ctl.q_full), 1);
    mbar_init(smem_u32(&ctl.q_empty), 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&ctl.full[i]), 1);
      mbar_init(smem_u32(&ctl.empty[i]), 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(smem_u32(&ctl.s_full[h]), 1);
      mbar_init(smem_u32(&ctl.p_full[h][0]), 4);  // one arrival a softmax warp
      mbar_init(smem_u32(&ctl.p_full[h][1]), 4);
      mbar_init(smem_u32(&ctl.o_full[h]), 1);
      mbar_init(smem_u32(&ctl.o_free[h]), 4);
      mbar_init(smem_u32(&ctl.clean[h]), 8);
    }
    mbar_init(smem_u32(&ctl.done), 1);
    ctl.abort = 0;
    ctl.poison = 0;
    mbar_init_fence();
    prefetch_map(&q_map);
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }
  wait_for_producer();
  release_dependents();  // the joining kernel waits for this one's completion by itself
  // the part of this CTA (the barriers inside also cover the set-up above)
  const PartialSums<2 * kRows, kDim> partials(a.workspace, gridDim.x);
  Walk w;
  {
    PlanPlace place;
    const bool has_part = plan_part<kThreads>(
        a.batch, a.status, gridDim.x, ctl.plan, [&](const PagedSequence& seq) { return chunk_units(c, seq); }, place);
    if (!has_part) {
      if (tid == 0) leave_join_tile(partials.tiles, nullptr, 0, 0, 0, 0);
      return;
    }
    const int step = 2 * c.half_tokens;
    const int64_t begin = place.cut.begin(blockIdx.x);
    int64_t before;
    w.t = plan_find<kThreads>(
        (place.seq.q_len + step - 1) / step, begin - place.before, ctl.plan,
        [&](int t) {
          return static_cast<int64_t>(chunk_tile(place.seq.q_len, place.seq.kv_len, step, window, t).blocks) *
                 a.cache.kv_heads;
        },
        before);
    w.s = place.sequence;
    w.seq = place.seq;
    w.left = place.cut.begin(blockIdx.x + 1) - begin;
    const int blocks = chunk_tile(w.seq.q_len, w.seq.kv_len, step, window, w.t).blocks;
    const int64_t rest = begin - place.before - before;
    w.kv_head = static_cast<int>(PlanCut::divide(rest, blocks));
    w.block = static_cast<int>(rest - static_cast<int64_t>(w.kv_head) * blocks);
    walk_tile(w, c);
    if (tid == 0) leave_join_tile(partials.tiles, &place, w.t, w.kv_head, begin - w.block, blocks);
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)),
                 "r"(kTmemColumns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = ctl.tmem_base;
  const int group = a.query_heads / a.cache.kv_heads;
  const int half_tokens = c.half_tokens;
  // Ring item 2n is K of the part's n-th block, item 2n + 1 its V: stage item % 4, phase item / 4.
  auto stage_of = [](uint32_t item) { return item % kStages; };
  auto phase_of = [](uint32_t item) { return (item / kStages) & 1; };
  auto wait = [&](uint64_t& bar, uint32_t phase) {
    if (!mbar_try(smem_u32(&bar), phase)) mbar_wait_or_abort(smem_u32(&bar), phase, &ctl.abort, a.status);
    __syncwarp();
  };

  if (warp == 8) {
    // ------------------------------------------------------------------------------------- TMA
    // The whole warp goes on or stops. A barrier is armed again only after its last load has landed, whatever
    // the MMA warp waited for: it runs on after a wait that gave up.
    bool ok = true;
    auto freed = [&](uint64_t& empty, uint64_t& full, uint32_t phase) {
      return __all_sync(0xffffffffu, mbar_wait_called(smem_u32(&empty), phase, &ctl.abort) &&
                                         mbar_wait_called(smem_u32(&full), phase, &ctl.abort)) != 0;
    };
    const int page_rows = min(1 << a.cache.page_shift, kChunkBlock);
    const int boxes = kChunkBlock / page_rows * kHalves;
    const int my_page = lane / kHalves;  // the lane's box: page and 64-wide half
    const int my_half = lane - my_page * kHalves;
    uint32_t item = 0;
    uint32_t segment = 0;
    do {
      if (segment > 0 && !freed(ctl.q_empty, ctl.q_full, (segment - 1) & 1)) {
        ok = false;
        break;
      }
      const int first_token = w.t * 2 * half_tokens;
      const int q_halves = first_token + half_tokens < w.seq.q_len ? 2 : 1;
      const uint32_t q_bar = smem_u32(&ctl.q_full);
      if (lane == 0) mbar_expect_tx(q_bar, q_halves * kHalves * half_tokens * group * 128);
      __syncwarp();
      if (lane < q_halves * kHalves) {
        const int half = lane / kHalves;
        const int column = lane - half * kHalves;
        tma_load_3d(q_smem + half * kOperand + column * kHalfBytes, &q_map, column * 64, w.kv_head * group,
                    w.seq.q_begin + first_token + half * half_tokens, q_bar);
      }
      ++segment;
      const int key_end = w.tile.last_position + 1;
      auto page_at = [&](int b) {  // the lane's page of block b, -1 when no row needs it
        const int key = (w.tile.block_begin + b) * kChunkBlock + my_page * page_rows;
        if (lane >= boxes || key >= key_end || key + page_rows <= w.tile.first_key) return -1;
        return paged_page(a.cache, a.batch, w.s, key >> a.cache.page_shift, a.status);
      };
      int page = page_at(w.block);
      for (int i = 0; i < w.count; ++i) {
        const int following = i + 1 < w.count ? page_at(w.block + i + 1) : -1;  // hides behind the waits
        const uint32_t loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
        const int key = (w.tile.block_begin + w.block + i) * kChunkBlock + my_page * page_rows;
        const int row = ((page * a.cache.kv_heads + w.kv_head) << a.cache.page_shift) +
                        (key & ((1 << a.cache.page_shift) - 1));
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++item) {
          const uint32_t stage = stage_of(item);
          if ((item >= kStages && !freed(ctl.empty[stage], ctl.full[stage], phase_of(item) ^ 1)) ||
              item >> 1 >= a.self_test_blocks) {
            ok = false;
            break;
          }
          const uint32_t bar = smem_u32(&ctl.full[stage]);
          if (lane == 0) mbar_expect_tx(bar, loads * page_rows * 128);
          __syncwarp();
          if (page >= 0) {
            tma_load_2d(ring + stage * kOperand + my_half * kHalfBytes + my_page * page_rows * 128,
                        kv == 0 ? &k_map : &v_map, my_half * 64, row, bar);
          }
        }
        if (!ok) break;
        page = following;
      }
    } while (ok && walk_next(w, c));
    if (!ok && item >> 1 < a.self_test_blocks && lane == 0) {
      report_status(a.status, kStatusWaitTimeout);
      ctl.abort = 1;
    }
    // the loads in flight land before the shared memory is released, even if the MMA warp no longer waits for them
    if (segment > 0) mbar_wait_called(smem_u32(&ctl.q_full), (segment - 1) & 1, nullptr);
    for (uint32_t i = item > kStages ? item - kStages : 0; i < item; ++i) {
      mbar_wait_called(smem_u32(&ctl.full[stage_of(i)]), phase_of(i), nullptr);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------------- MMA
    // The halves' products are issued in turn, [O += P V, next S] of half 0, then of half 1, which keeps
    // the halves half a block apart: with a warp for each half they fell into step, their exponentials
    // sharing the SFU and their products the tensor pipe (985 against 880 us for two 4K chunks).
    const uint32_t elected = elect_one();
    uint32_t turn = 0;  // blocks so far
    uint32_t segment = 0;
    uint32_t cleaned = 0;  // the next phases of the two `clean` barriers, a bit each
    do {
      int begin0, end0, begin1, end1;
      w.half_range(0, half_tokens, window, begin0, end0);
      w.half_range(1, half_tokens, window, begin1, end1);
      const int end = w.block + w.count;
      auto needs = [&](int half, int b) { return half == 0 ? b >= begin0 && b < end0 : b >= begin1 && b < end1; };
      // S = Q K^T of block b (the n-th of the part) where the half needs it
      auto scores = [&](int half, int b, uint32_t n) {
        if (needs(half, b)) {
          const uint64_t q_at = desc_k_major(q_smem + half * kOperand);
          const uint64_t k_at = desc_k_major(ring + stage_of(2 * n) * kOperand);
#pragma unroll
          for (int k = 0; k < kDim / 16; ++k) {  // 16 values, 32 bytes of a row, a step
            const uint64_t offset = (k >> 2) * (kHalfBytes >> 4) + (k & 3) * 2;
            mma_ss(elected, tmem + half * 128, q_at + offset, k_at + offset, c.idesc_s, k > 0 ? 1u : 0u);
          }
          mma_commit(elected, smem_u32(&ctl.s_full[half]));
        } else {
          mbar_arrive_if(elected, smem_u32(&ctl.s_full[half]));
        }
        if (half == 1) {
          mma_commit(elected, smem_u32(&ctl.empty[stage_of(2 * n)]));
          if (b == end - 1) mma_commit(elected, smem_u32(&ctl.q_empty));  // Q has been read for the last time
        }
      };
      auto wait_k = [&](uint32_t n) {
        wait(ctl.full[stage_of(2 * n)], phase_of(2 * n));
        fence_after();
      };
      wait(ctl.q_full, segment & 1);
      wait_k(turn);
      scores(0, w.block, turn);
      scores(1, w.block, turn);
      uint32_t waited_o = segment == 0 ? 3u : 0u;  // halves whose O of the last segment has been read
      for (int b = w.block; b < end; ++b, ++turn) {
        const uint32_t v_item = 2 * turn + 1;
        const uint32_t stage = stage_of(v_item);
        wait(ctl.full[stage], phase_of(v_item));
        if (!w.whole(b, window)) {  // V of this block is cleared by the softmax warps first
          wait(ctl.clean[turn & 1], (cleaned >> (turn & 1)) & 1);
          cleaned ^= 1u << (turn & 1);
        }
        const uint64_t v_at = desc_mn_major(ring + stage * kOperand, kHalfBytes);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bool needed = needs(half, b);
          if (needed && !(waited_o >> half & 1)) {
            wait(ctl.o_free[half], (segment - 1) & 1);
            waited_o |= 1u << half;
          }
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            // a wait behind MMAs stalls until they have drained, so the next K is waited for up here
            if (half == 0 && part == 1 && b + 1 < end) wait_k(turn + 1);
            wait(ctl.p_full[half][part], turn & 1);
            fence_after();
            if (needed) {
              const bool first = b == (half == 0 ? begin0 : begin1);
#pragma unroll
              for (int k = part * 6; k < 6 + part * 2; ++k) {  // 16 keys a step
                mma_ts(elected, tmem + kTmemO + half * 128, tmem + half * 128 + k * 8, v_at + k * (16 * 128 >> 4),
                       c.idesc_o, first && k == 0 ? 0u : 1u);
              }
              if (part == 1) mma_commit(elected, smem_u32(&ctl.o_full[half]));
            }
          }
          if (half == 1) mma_commit(elected, smem_u32(&ctl.empty[stage]));
          if (b + 1 < end) scores(half, b + 1, turn + 1);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!(waited_o >> half & 1)) wait(ctl.o_free[half], (segment - 1) & 1);
        // a half without blocks takes part too, so that its softmax warps stay within a segment of it
        if ((half == 0 ? begin0 == end0 : begin1 == end1)) mbar_arrive_if(elected, smem_u32(&ctl.o_full[half]));
      }
      ++segment;
    } while (walk_next(w, c));
    // every MMA has completed before TMEM and shared memory are released
    mma_commit(elected, smem_u32(&ctl.done));
    mbar_wait_called(smem_u32(&ctl.done), 0, nullptr);
  } else {
    // --------------------------------------------------------------------------------- softmax
    const int half = warp >> 2;
    const int row = tid & (kRows - 1);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + half * 128 + lane_base;
    const uint32_t o_tmem = tmem + kTmemO + half * 128 + lane_base;
    const int row_token = row / group;
    const int row_head = row - row_token * group;
    uint32_t turn = 0;
    const uint32_t elected = lane == 0 ? 1u : 0u;
    uint32_t outputs = 0;  // phases of o_full so far: one a block, one a segment without any
    uint32_t segment = 0;
    uint32_t cleaned = 0;       // the next phases of the two `clean` barriers, a bit each
    uint32_t cleaned_once = 0;  // which of them have had one
    do {
      int h_begin, h_end;
      w.half_range(half, half_tokens, window, h_begin, h_end);
      const int end = w.block + w.count;
      const int token = w.t * 2 * half_tokens + half * half_tokens + row_token;
      const bool row_in = row_token < half_tokens && token < w.seq.q_len;
      const int position = w.seq.kv_len - w.seq.q_len + token;
      const int row_first = window > 0 && position >= window ? position - window + 1 : 0;
      const int row_last = row_in ? position : -1;
      if (tid == 0) atomicAnd(&ctl.poison, ~(1u << ((segment + 16) & 31)));  // the halves are never 16 segments apart
      float reference = -INFINITY;
      float l = 0.0f;
      // tcgen05.ld / tcgen05.st are warp-collective: every branch around them is uniform per warp
      for (int b = w.block; b < end; ++b, ++turn) {
        const bool needed = b >= h_begin && b < h_end;
        const bool whole = w.whole(b, window);
        const int key0 = (w.tile.block_begin + b) * kChunkBlock;
        // every block passes through s_full and p_full, needed by the half or not, so that neither side
        // is ever more than one phase ahead of a barrier that it waits on
        wait(ctl.s_full[half], turn & 1);
        if (!whole) {
          // Clear what no row of the tile sees, and values that are not finite (a probability of zero
          // times one would be NaN); the rows that see those get them added at the end.
          const uint32_t v_item = 2 * turn + 1;
          wait(ctl.full[stage_of(v_item)], phase_of(v_item));
          uint4* v = reinterpret_cast<uint4*>(smem + Layout<kDim>::kRing + stage_of(v_item) * kOperand);
          bool bad = false;
#pragma unroll 4
          for (int i = tid; i < static_cast<int>(kOperand / 16); i += 2 * kRows) {
            const int key = key0 + ((i >> 3) & (kChunkBlock - 1));  // eight chunks of 16 bytes a row
            if (key < w.tile.first_key || key > w.tile.last_position) {
              v[i] = make_uint4(0u, 0u, 0u, 0u);
              continue;
            }
            uint4 value = v[i];
            if (nonfinite_pair<T>(value.x) | nonfinite_pair<T>(value.y) | nonfinite_pair<T>(value.z) |
                nonfinite_pair<T>(value.w)) {
              bad = true;
              value.x = finite_pair<T>(value.x);
              value.y = finite_pair<T>(value.y);
              value.z = finite_pair<T>(value.z);
              value.w = finite_pair<T>(value.w);
              v[i] = value;
            }
          }
          __syncwarp();
          if (bad) atomicOr(&ctl.poison, 1u << (segment & 31));
          fence_async_shared();
          __syncwarp();
          mbar_arrive_if(elected, smem_u32(&ctl.clean[turn & 1]));
          cleaned ^= 1u << (turn & 1);
          cleaned_once |= 1u << (turn & 1);
        }
        if (!needed) {
          mbar_arrive_if(elected, smem_u32(&ctl.p_full[half][0]));
          mbar_arrive_if(elected, smem_u32(&ctl.p_full[half][1]));
          continue;
        }
        fence_after();
        // S passes through the registers twice, 32 columns a time: C D A B for the maximum, A B (still
        // there) C D for the probabilities, whose loads hide behind the exponentials before them. P's
        // 16-bit pairs take the place of scores already read. The products with V start when A B C are
        // there, so that those of D alone stand between the last probability and the next scores.
        const int low = row_first - key0;
        const int high = row_last - key0;
        uint32_t x[2][32];
        auto mask = [&](uint32_t (&v)[32], int column) {
          if (__builtin_expect(whole, 1)) return;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i + column > high || i + column < low) v[i] = __float_as_uint(-INFINITY);
          }
        };
        float top[kChains];
#pragma unroll
        for (int i = 0; i < kChains; ++i) top[i] = -INFINITY;
#pragma unroll 1
        for (int column = 64; column >= 0; column -= 64) {
          tmem_ld32(s_tmem + column, x[0]);
          tmem_ld32(s_tmem + column + 32, x[1]);
          tmem_wait_ld();
          mask(x[0], column);
          mask(x[1], column + 32);
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            top[(i / 2) % kChains] = max3(top[(i / 2) % kChains], __uint_as_float(x[i >> 5][i & 31]),
                                          __uint_as_float(x[i >> 5][(i & 31) + 1]));
          }
        }
        const float block_top = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2;
        // the row's reference moves only when the block's maximum exceeds it by more than its reach (rounded
        // down, so that no score passes further), so O is rarely rescaled
        const bool move = block_top > __fadd_rd(reference, kReferenceReach<T>);
        const float moved = block_top - kReferenceBelow<T>;
        const bool rescale = move && reference != -INFINITY;
        if (__any_sync(0xffffffffu, rescale)) {
          // O holds the segment's blocks before this one
          wait(ctl.o_full[half], (outputs - 1) & 1);
          fence_after();
          const float factor = rescale ? ex2_ftz(reference - moved) : 1.0f;
#pragma unroll 1
          for (int i = 0; i < kDim / 32; ++i) {
            uint32_t raw[32];
            tmem_ld32(o_tmem + i * 32, raw);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = __float_as_uint(__uint_as_float(raw[j]) * factor);
            tmem_st32(o_tmem + i * 32, raw);
          }
          l *= factor;
        }
        if (move) reference = moved;
        const float base = reference == -INFINITY ? 0.0f : -reference;
        const unsigned long long scale2 = pack_f32x2(a.scale_log2, a.scale_log2);
        const unsigned long long base2 = pack_f32x2(base, base);
        unsigned long long sums[kChains / 2];
#pragma unroll
        for (int i = 0; i < kChains / 2; ++i) sums[i] = 0ull;
        auto probabilities = [&](const uint32_t (&v)[32], uint32_t column) {
          uint32_t packed[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float p0, p1;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), scale2, base2),
                         p0, p1);
            p0 = ex2_ftz(p0);
            p1 = ex2_ftz(p1);
            sums[i % (kChains / 2)] = add_f32x2(sums[i % (kChains / 2)], pack_f32x2(p0, p1));
            packed[i] = pack2<T>(p0, p1);  // rounded: see kReferenceBelow
          }
          tmem_st16(s_tmem + column, packed);
        };
        // Rolled: the softmax and MMA warps of an SM quarter share an instruction cache that the unrolled
        // form does not fit (886 against 846 us for two 4K chunks; a quarter of the exponentials as
        // polynomials on the FMA pipe: 846 against 864 us, the same within the noise, and left out).
#pragma unroll 1
        for (int pair = 0; pair < 2; ++pair) {
          probabilities(x[0], pair * 32);
          if (pair == 0) {
            tmem_ld32(s_tmem + 64, x[0]);
          } else {
            tmem_wait_st();
            fence_before();
            mbar_arrive_if(elected, smem_u32(&ctl.p_full[half][0]));
            tmem_wait_ld();
            mask(x[1], 96);
          }
          probabilities(x[1], pair * 32 + 16);
          if (pair == 0) {
            tmem_wait_ld();
            tmem_ld32(s_tmem + 96, x[1]);
            mask(x[0], 64);
          }
        }
        tmem_wait_st();
        fence_before();
        mbar_arrive_if(elected, smem_u32(&ctl.p_full[half][1]));
#pragma unroll
        for (int i = 0; i < kChains / 2; ++i) {
          float s0, s1;
          unpack_f32x2(sums[i], s0, s1);
          l += s0 + s1;
        }
        ++outputs;
      }
      // ---- the segment's rows: O / l, or the partial sums
      const bool any = h_end > h_begin;
      if (!any) ++outputs;
      wait(ctl.o_full[half], (outputs - 1) & 1);
      fence_after();
      // every thread's share of the cleared blocks is done when their barriers' last phases are
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (cleaned_once >> i & 1) wait(ctl.clean[i], ((cleaned >> i) & 1) ^ 1);
      }
      const bool poisoned = (*reinterpret_cast<volatile unsigned*>(&ctl.poison) >> (segment & 31)) & 1;
      const bool begins = w.block == 0;
      const bool complete = begins && w.count == w.tile.blocks;
      const float factor = complete ? (l != 0.0f ? 1.0f / l : 0.0f) : 1.0f;
      const int head = w.kv_head * group + row_head;
      const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (begins ? 1 : 0);
      const int64_t out_token = w.seq.q_begin + token;
#pragma unroll 1
      for (int i = 0; i < kDim / 32; ++i) {
        uint32_t raw[32];
        __syncwarp();  // rows of a warp part below
        if (any) {
          tmem_ld32(o_tmem + i * 32, raw);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) raw[j] = 0u;
        }
        if (row_in && complete) {
          T* to = static_cast<T*>(a.out) + out_token * a.out_stride + head * kDim + i * 32;
          uint32_t packed[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            packed[j] = pack2<T>(__uint_as_float(raw[2 * j]) * factor, __uint_as_float(raw[2 * j + 1]) * factor);
          }
          *reinterpret_cast<uint4*>(to) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
          *reinterpret_cast<uint4*>(to + 8) = make_uint4(packed[4], packed[5], packed[6], packed[7]);
          *reinterpret_cast<uint4*>(to + 16) = make_uint4(packed[8], packed[9], packed[10], packed[11]);
          *reinterpret_cast<uint4*>(to + 24) = make_uint4(packed[12], packed[13], packed[14], packed[15]);
        } else if (row_in) {
          // [columns / 4][rows][4]: a warp's rows are neighbours
          float4* to = reinterpret_cast<float4*>(partials.sums) + slot * (2 * kRows) * (kDim / 4) +
                       i * 8 * (2 * kRows) + half * kRows + row;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            to[j * (2 * kRows)] = make_float4(__uint_as_float(raw[4 * j]), __uint_as_float(raw[4 * j + 1]),
                                __uint_as_float(raw[4 * j + 2]), __uint_as_float(raw[4 * j + 3]));
          }
        }
      }
      fence_before();
      __syncwarp();
      mbar_arrive_if(elected, smem_u32(&ctl.o_free[half]));
      if (row_in && poisoned) {
        add_nonfinite<T, kDim>(a, w, row_first, row_last,
                               complete ? static_cast<T*>(a.out) + out_token * a.out_stride + head * kDim : nullptr,
                               partials.sums + (slot * (2 * kRows) * (kDim / 4) + half * kRows + row) * 4);
      }
      if (row_in) {
        if (!complete) {
          partials.stats[slot * (2 * kRows) + half * kRows + row] = make_float2(reference, l);
        } else if (a.lse != nullptr) {
          a.lse[out_token * a.query_heads + head] = l != 0.0f ? reference + log2f(l) : -INFINITY;
        }
      }
      __syncwarp();
      ++segment;
    } while (walk_next(w, c));
  }

  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 8) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
  }
}

// Joins the parts of the tile that the beginning of part blockIdx.x + 1 cuts, in the order of the CTAs;
// blockIdx.y: kJoinRows of the tile's rows.
template <typename T, int kDim>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_chunk_join_kernel(const ChunkArgs c, int ctas) {
  // every thread waits, so that this grid does not complete before the one whose sums it reads
  wait_for_producer();
  release_dependents();
  const PagedAttentionArgs& a = c.a;
  const PartialSums<2 * kRows, kDim> partials(a.workspace, ctas);
  const JoinTile place = partials.tiles[blockIdx.x + 1];
  const int last = place.last;
  if (last < 0) return;
  const PagedSequence seq = place.seq;
  const int boundary = blockIdx.x;  // the part in which the tile begins
  const int group = a.query_heads / a.cache.kv_heads;
  constexpr int kBatch = 4;  // parts whose loads are in flight together
  // a warp takes 32 rows of eight columns
  const int tile_row = blockIdx.y * kJoinRows + (threadIdx.x & 31);
  const int half = tile_row / kRows;
  const int row = tile_row - half * kRows;
  const int row_token = row / group;
  const int token = (place.tile * 2 + half) * c.half_tokens + row_token;
  if (row_token >= c.half_tokens || token >= seq.q_len) return;
  const int head = place.kv_head * group + row - row_token * group;
  for (int column = (threadIdx.x >> 5) * 8; column < kDim; column += kJoinThreads / 32 * 8) {
    float top = -INFINITY;
    float sum = 0.0f;
    float o[8] = {};
    for (int first = boundary; first <= last; first += kBatch) {
      float2 stats[kBatch];
      float4 piece[kBatch][2];
      float high = top;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int part = first + i;
        stats[i] = make_float2(-INFINITY, 0.0f);
        piece[i][0] = piece[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (part <= last) {
          const int64_t slot = static_cast<int64_t>(part) * 2 + (part == boundary ? 1 : 0);
          const float4* from = reinterpret_cast<const float4*>(partials.sums) + slot * (2 * kRows) * (kDim / 4) +
                               column / 4 * (2 * kRows) + tile_row;
          stats[i] = partials.stats[slot * (2 * kRows) + tile_row];
          piece[i][0] = from[0];
          piece[i][1] = from[2 * kRows];
        }
        high = fmaxf(high, stats[i].x);
      }
      const float keep = top == -INFINITY ? 0.0f : ex2_ftz(top - high);
      sum *= keep;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= keep;
      top = high;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float factor = stats[i].x == -INFINITY ? 0.0f : ex2_ftz(stats[i].x - top);
        sum += factor * stats[i].y;
        const float values[8] = {piece[i][0].x, piece[i][0].y, piece[i][0].z, piece[i][0].w,
                                 piece[i][1].x, piece[i][1].y, piece[i][1].z, piece[i][1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += factor * values[j];
      }
    }
    const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] *= inverse;
    T* to = static_cast<T*>(a.out) + (seq.q_begin + token) * a.out_stride + head * kDim + column;
    *reinterpret_cast<uint4*>(to) = pack8<T>(o);
    if (column == 0 && a.lse != nullptr) {
      a.lse[static_cast<int64_t>(seq.q_begin + token) * a.query_heads + head] =
          sum != 0.0f ? top + log2f(sum) : -INFINITY;
    }
  }
}

template <typename T>
bool encode_map(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                const cuuint32_t* box) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint32_t element_strides[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(map, type, rank, const_cast<void*>(base), dims, strides, box, element_strides,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int kDim>
cudaError_t launch_chunk(const PagedAttentionArgs& a, int few, cudaStream_t stream) {
  static_assert(Layout<kDim>::bytes() <= 227 * 1024, "one CTA's shared memory");
  int device = 0;
  cudaGetDevice(&device);
  static DeviceOnce configured;  // the shared-memory opt-in is a per-device attribute
  const cudaError_t opted = configured.run(device, [] {
    return cudaFuncSetAttribute(paged_attention_chunk_kernel<T, kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(Layout<kDim>::bytes()));
  });
  if (opted != cudaSuccess) return opted;
  const int group = a.query_heads / a.cache.kv_heads;
  ChunkArgs c;
  c.a = a;
  c.half_tokens = kRows / group;
  c.few = few;
  const uint32_t format = std::is_same_v<T, __half> ? 0u : 1u;
  c.idesc_s = idesc(format, false, kChunkBlock);
  c.idesc_o = idesc(format, true, kDim);
  CUtensorMap q_map, k_map, v_map;
  // Q: (64 values, the group's heads, half a tile's tokens); rows past the call's are zeros
  const cuuint64_t q_dims[3] = {kDim, static_cast<cuuint64_t>(a.query_heads), static_cast<cuuint64_t>(a.batch.tokens)};
  const cuuint64_t q_strides[2] = {kDim * 2, static_cast<cuuint64_t>(a.q_stride) * 2};
  const cuuint32_t q_box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(c.half_tokens)};
  const cuuint64_t pool_rows = (static_cast<cuuint64_t>(a.cache.page_count) * a.cache.kv_heads) << a.cache.page_shift;
  const cuuint64_t dims[2] = {kDim, pool_rows};
  const cuuint64_t strides[1] = {kDim * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(std::min(1 << a.cache.page_shift, kChunkBlock))};
  if (!encode_map<T>(&q_map, 3, a.q, q_dims, q_strides, q_box) ||
      !encode_map<T>(&k_map, 2, a.cache.k_pages, dims, strides, box) ||
      !encode_map<T>(&v_map, 2, a.cache.v_pages, dims, strides, box)) {
    return cudaErrorInvalidValue;
  }
  const int ctas = sm_count();
  const cudaError_t status = launch_overlapped(paged_attention_chunk_kernel<T, kDim>, dim3(ctas), dim3(kThreads),
                                               Layout<kDim>::bytes(), stream, q_map, k_map, v_map, c);
  if (status != cudaSuccess || ctas < 2) return status;
  return launch_overlapped(paged_attention_chunk_join_kernel<T, kDim>, dim3(ctas - 1, 2 * kRows / kJoinRows),
                           dim3(kJoinThreads), 0, stream, c, ctas);
}

}  // namespace

int64_t paged_attention_chunk_workspace(int head_dim) { return partial_bytes(2 * kRows, head_dim, sm_count()); }

cudaError_t launch_paged_attention_chunk(const PagedAttentionArgs& a, int few, cudaStream_t stream) {
  if (a.cache.dtype == kActFp16) {
    return a.cache.head_dim == 128 ? launch_chunk<__half, 128>(a, few, stream) : launch_chunk<__half, 64>(a, few, stream);
  }
  return a.cache.head_dim == 128 ? launch_chunk<__nv_bfloat16, 128>(a, few, stream)
                                 : launch_chunk<__nv_bfloat16, 64>(a, few, stream);
}

}  // namespace arb
