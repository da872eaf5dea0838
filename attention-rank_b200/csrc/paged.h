// Serving operators: launchers of the scaled rotary table and rotation (rotary.cu), the append to a
// paged KV cache (paged_append.cu) and the attention over it
// (paged_attention.cu, paged_attention_tc.cu). All pointers are
// device pointers; all launches are asynchronous on `stream`. The contracts are those of
// include/attnrank_b200.h; argument checks are in capi_paged.cu.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"

namespace arb {

constexpr int kMaxTableFrequencies = 256;  // rotary_dim / 2 of the largest table

// Turns a position (frequency / 2 pi) of every pair, passed by value.
struct TableTurns {
  double value[kMaxTableFrequencies];
};

cudaError_t launch_rope_table_scaled(const TableTurns& turns, int half, float multiplier, int positions,
                                     float* cos_table, float* sin_table, cudaStream_t stream);

struct RotaryArgs {
  const void* x = nullptr;
  int64_t x_token_stride = 0;  // elements
  int64_t x_head_stride = 0;
  void* out = nullptr;
  int64_t out_token_stride = 0;
  int64_t out_head_stride = 0;
  const int32_t* positions = nullptr;
  int tokens = 0;
  int heads = 0;
  int head_dim = 0;
  int rotary_dim = 0;
  int interleaved = 0;
  int inverse = 0;
  const float* cos_table = nullptr;
  const float* sin_table = nullptr;
  int table_positions = 0;
  int* status = nullptr;
  int dtype = kActFp16;
};
cudaError_t launch_rotary_positions(const RotaryArgs& args, cudaStream_t stream);

struct PagedCache {
  void* k_pages = nullptr;  // 16-bit [page_count][kv_heads][page_size][head_dim]
  void* v_pages = nullptr;
  int page_count = 0;
  int page_shift = 0;  // log2(page_size)
  int kv_heads = 0;
  int head_dim = 0;
  int dtype = kActFp16;
};

struct PagedBatch {
  int sequences = 0;
  int tokens = 0;
  int max_query = 0;
  int table_stride = 0;
  int capacity = 0;  // cached tokens a page-table row can describe
  const int32_t* q_offsets = nullptr;
  const int32_t* kv_lengths = nullptr;
  const int32_t* page_table = nullptr;
};

struct PagedAppendArgs {
  PagedCache cache;
  PagedBatch batch;
  const void* qkv = nullptr;
  int64_t qkv_stride = 0;
  const float* bias = nullptr;
  int query_heads = 0;  // heads of the qkv row
  void* q_out = nullptr;
  int64_t q_out_stride = 0;
  const float* cos_table = nullptr;
  const float* sin_table = nullptr;
  int table_positions = 0;
  int rotary_dim = 0;
  int interleaved = 0;
  int* status = nullptr;
};
cudaError_t launch_paged_append(const PagedAppendArgs& args, cudaStream_t stream);

struct PagedAttentionArgs {
  PagedCache cache;
  PagedBatch batch;
  const void* q = nullptr;
  int64_t q_stride = 0;
  int query_heads = 0;
  float scale_log2 = 0.0f;  // score scale times log2(e)
  int sliding_window = 0;
  void* out = nullptr;
  int64_t out_stride = 0;
  float* lse = nullptr;
  void* workspace = nullptr;
  int* status = nullptr;
  uint32_t self_test_blocks = ~0u;  // key blocks of its part that a CTA loads; the waits for more run out
};
int64_t paged_attention_workspace(const PagedCache& cache, const PagedBatch& batch, int query_heads);
cudaError_t launch_paged_attention(const PagedAttentionArgs& args, cudaStream_t stream);
// The form for more than a few rows a KV head (paged_attention_tc.cu).
int64_t paged_attention_chunk_workspace(int head_dim);
// It leaves out sequences of at most `few` new tokens.
cudaError_t launch_paged_attention_chunk(const PagedAttentionArgs& args, int few, cudaStream_t stream);

// ------------------------------------------------------------------------------ device helpers
#ifdef __CUDACC__

// The probabilities 2^(x - reference) are rounded to the 16-bit type for the product with V: the tensor
// cores take both operands in one type, and two products for a split probability would double the work.
// A row's reference is set kReferenceBelow under its maximum and moves when a score exceeds it by more than
// kReferenceReach, so a probability stays below 2^15 in fp16 and 2^8 in bf16. In fp16 that leaves weights
// down to 2^-21 of the largest one with all their bits; with a reference at the maximum itself it was 2^-14,
// and 2^17 keys of 2^-25.5 each, 1/362 of the row together, vanished.
template <typename T>
constexpr float kReferenceBelow = std::is_same_v<T, __half> ? 7.0f : 0.0f;  // log2 units
template <typename T>
constexpr float kReferenceReach = kReferenceBelow<T> + 8.0f;

// The batch's arrays are read through L2 (__ldcg): a kernel launched ahead of its producer's end must not
// find an older copy of them in the read-only cache.

// One sequence of a batch; q_len == 0 when it has no new tokens or its metadata is out of range
// (which is reported).
struct PagedSequence {
  int q_begin;
  int q_len;
  int kv_len;
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch& b, int s, int* status) {
  const int begin = __ldcg(b.q_offsets + s);
  const int end = __ldcg(b.q_offsets + s + 1);
  const int length = __ldcg(b.kv_lengths + s);
  const bool ok = begin >= 0 && end >= begin && end <= b.tokens && end - begin <= b.max_query && length >= 0 &&
                  length <= b.capacity;
  if (!ok) {
    report_status(status, kStatusPagedBatch);
    return {0, 0, 0};
  }
  return {begin, end - begin, length};
}

// Where `token` lies among the offsets: the sequence whose rows hold it if they never decrease, else any
// sequence or -1. The whole warp calls it with the same token. Each round probes 32 evenly spaced
// offsets, so 1024 sequences take two dependent loads.
__device__ __forceinline__ int paged_search(const PagedBatch& b, int token) {
  const int lane = threadIdx.x & 31;
  int low = 0;
  int count = b.sequences + 1;  // offsets not yet known to be above or not above `token`
  while (count > 0) {
    const int step = (count + 31) >> 5;
    const int at = (lane + 1) * step - 1;
    const bool not_above = at < count && __ldcg(b.q_offsets + low + at) <= token;
    const int passed = __popc(__ballot_sync(0xffffffffu, not_above)) * step;
    low += passed;
    count = max(0, min(step - 1, count - passed));
  }
  return low >= 1 && low <= b.sequences ? low - 1 : -1;
}

// The sequence whose rows hold `token` and that is in range (`seq`), or -1; the whole warp calls it with
// the same token. Offsets that decrease somewhere mislead the search, so where it finds no such sequence,
// though an offset lies behind the token, every one is looked at.
__device__ __forceinline__ int paged_sequence_of(const PagedBatch& b, int token, int* status, PagedSequence& seq) {
  const int lane = threadIdx.x & 31;
  const int found = paged_search(b, token);
  bool behind = false;
  if (found >= 0) {
    seq = paged_sequence(b, found, status);
    if (token >= seq.q_begin && token - seq.q_begin < seq.q_len) return found;
    behind = true;
  } else {
    // eight loads in flight: a row of padding waits for one round of them, not for each
    for (int at = lane; at <= b.sequences; at += 256) {
#pragma unroll
      for (int i = 0; i < 8; ++i) behind |= __ldcg(b.q_offsets + min(at + 32 * i, b.sequences)) > token;
    }
  }
  if (!__any_sync(0xffffffffu, behind)) return -1;  // rows behind the last sequence
  for (int base = 0; base < b.sequences; base += 32) {
    if (base + lane < b.sequences) seq = paged_sequence(b, base + lane, status);
    const bool holds = base + lane < b.sequences && token >= seq.q_begin && token - seq.q_begin < seq.q_len;
    const unsigned holders = __ballot_sync(0xffffffffu, holds);
    if (holders != 0) {
      const int owner = __ffs(holders) - 1;
      seq.q_begin = __shfl_sync(0xffffffffu, seq.q_begin, owner);
      seq.q_len = __shfl_sync(0xffffffffu, seq.q_len, owner);
      seq.kv_len = __shfl_sync(0xffffffffu, seq.kv_len, owner);
      return base + owner;
    }
  }
  return -1;
}

// A page id of sequence s, clamped into the pool (an id outside it is reported).
__device__ __forceinline__ int paged_page(const PagedCache& c, const PagedBatch& b, int s, int index, int* status) {
  const int page = __ldcg(b.page_table + static_cast<int64_t>(s) * b.table_stride + index);
  if (page >= 0 && page < c.page_count) return page;
  report_status(status, kStatusPagedBatch);
  return 0;
}

template <bool kInterleaved>
__device__ __forceinline__ void rotate16(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8]) {
  if constexpr (kInterleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
      a[2 * i] = a0 * c[i] - a1 * s[i];
      a[2 * i + 1] = a1 * c[i] + a0 * s[i];
      b[2 * i] = b0 * c[4 + i] - b1 * s[4 + i];
      b[2 * i + 1] = b1 * c[4 + i] + b0 * s[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  }
}

// Sixteen values of a head as eight rotation pairs, rotated in place: in the half layout pair i is
// (low[i], high[i]); interleaved, low and high are sixteen consecutive values and pair i is values
// 2i and 2i + 1 of them.
template <typename T, bool kInterleaved>
__device__ __forceinline__ void rotate16(uint4& low, uint4& high, const float (&c)[8], const float (&s)[8]) {
  float a[8], b[8];
  unpack8<T>(low, a);
  unpack8<T>(high, b);
  rotate16<kInterleaved>(a, b, c, s);
  low = pack8<T>(a);
  high = pack8<T>(b);
}

#endif  // __CUDACC__

}  // namespace arb
