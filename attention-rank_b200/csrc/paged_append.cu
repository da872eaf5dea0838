// Append of new tokens to a paged KV cache with the rotation on the way (contract in
// include/attnrank_b200.h): one read of each q|k|v value and one write of it to its place, so HBM bounds
// it (11.5K tokens of 48 heads x 128: 51 us a call, 0.86 of the measured copy).
#include <algorithm>

#include "common.cuh"
#include "layer_kernels.h"
#include "paged.h"

namespace arb {
namespace {

constexpr int kThreads = 256;

// One CTA takes kTokens consecutive rows. A warp finds each row's sequence, position and page slot
// once; then the CTA walks the items (row, kHeads heads, 16 values of each head), rotation pairs
// first, as in rotary.cu.
template <typename T, bool kInterleaved, bool kBias, int kHeads, int kTokens>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedAppendArgs a, int first_head, int units,
                                                                int rotated_units, int groups) {
  static_assert(kTokens < kThreads / 32, "one warp finds each row's place, another checks the batch");
  __shared__ int position_of[kTokens];
  __shared__ int64_t slot_of[kTokens];
  const int begin = blockIdx.x * kTokens;
  const int warp = threadIdx.x >> 5;
  if (warp < kTokens) {
    const int token = begin + warp;
    int position = -1;
    int64_t slot = 0;
    PagedSequence seq{0, 0, 0};
    const int s = token < a.batch.tokens ? paged_sequence_of(a.batch, token, a.status, seq) : -1;
    if (s >= 0) {
      position = seq.kv_len - seq.q_len + token - seq.q_begin;
      if (position >= 0 && a.rotary_dim > 0 && position >= a.table_positions) {
        report_status(a.status, kStatusPositionOutOfRange);
        position = -1;
      }
      if (position >= 0) {
        const int index = position >> a.cache.page_shift;
        const int page = __ldcg(a.batch.page_table + static_cast<int64_t>(s) * a.batch.table_stride + index);
        if (page >= 0 && page < a.cache.page_count) {
          const int in_page = position & ((1 << a.cache.page_shift) - 1);
          slot = (static_cast<int64_t>(page) * a.cache.kv_heads << a.cache.page_shift) + in_page;
        } else {
          report_status(a.status, kStatusPagedBatch);
          position = -1;
        }
      }
    }
    if ((threadIdx.x & 31) == 0) {
      position_of[warp] = position;
      slot_of[warp] = slot;
    }
  } else if (warp == kTokens) {  // sequences out of range are reported even where no row leads to them
    for (int64_t s = blockIdx.x * 32 + (threadIdx.x & 31); s < a.batch.sequences; s += gridDim.x * 32) {
      paged_sequence(a.batch, static_cast<int>(s), a.status);
    }
  }
  __syncthreads();
  const int head_dim = a.cache.head_dim;
  const int heads = a.query_heads + 2 * a.cache.kv_heads;
  const int rotated_heads = a.query_heads + a.cache.kv_heads;
  const int per_token = groups * units;
  for (int item = threadIdx.x; item < kTokens * per_token; item += kThreads) {
    const int row = item / per_token;
    const int rest = item - row * per_token;
    const int group = rest / units;
    const int unit = rest - group * units;
    const int position = position_of[row];
    if (position < 0) continue;
    const int64_t token = begin + row;
    const bool rotated = unit < rotated_units;
    int low_at, high_at;
    if (!rotated) {
      low_at = a.rotary_dim + (unit - rotated_units) * 16;
      high_at = low_at + 8;
    } else if (kInterleaved) {
      low_at = unit * 16;
      high_at = low_at + 8;
    } else {
      low_at = unit * 8;
      high_at = (a.rotary_dim >> 1) + unit * 8;
    }
    const int first = first_head + group * kHeads;
    const T* x = static_cast<const T*>(a.qkv) + token * a.qkv_stride;
    uint4 low[kHeads], high[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (first + h < heads) {
        low[h] = *reinterpret_cast<const uint4*>(x + (first + h) * head_dim + low_at);
        high[h] = *reinterpret_cast<const uint4*>(x + (first + h) * head_dim + high_at);
      }
    }
    float c[8], s[8];
    if (rotated && first < rotated_heads) {
      const int64_t at = static_cast<int64_t>(position) * (a.rotary_dim >> 1) + unit * 8;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(a.cos_table + at + i));
        const float4 s4 = __ldg(reinterpret_cast<const float4*>(a.sin_table + at + i));
        c[i] = c4.x, c[i + 1] = c4.y, c[i + 2] = c4.z, c[i + 3] = c4.w;
        s[i] = s4.x, s[i + 1] = s4.y, s[i + 2] = s4.z, s[i + 3] = s4.w;
      }
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const int head = first + h;
      if (head >= heads) break;
      const bool turn = rotated && head < rotated_heads;
      if (kBias || turn) {
        float lo[8], hi[8];
        unpack8<T>(low[h], lo);
        unpack8<T>(high[h], hi);
        if constexpr (kBias) {
          const float* b = a.bias + head * head_dim;
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const float4 b0 = __ldg(reinterpret_cast<const float4*>(b + low_at + i));
            const float4 b1 = __ldg(reinterpret_cast<const float4*>(b + high_at + i));
            lo[i] += b0.x, lo[i + 1] += b0.y, lo[i + 2] += b0.z, lo[i + 3] += b0.w;
            hi[i] += b1.x, hi[i + 1] += b1.y, hi[i + 2] += b1.z, hi[i + 3] += b1.w;
          }
        }
        if (turn) rotate16<kInterleaved>(lo, hi, c, s);
        low[h] = pack8<T>(lo);
        high[h] = pack8<T>(hi);
      }
      T* out;
      if (head < a.query_heads) {
        out = static_cast<T*>(a.q_out) + token * a.q_out_stride + head * head_dim;
      } else {
        const bool is_key = head < rotated_heads;
        const int kv_head = head - (is_key ? a.query_heads : rotated_heads);
        out = static_cast<T*>(is_key ? a.cache.k_pages : a.cache.v_pages) +
              (slot_of[row] + (static_cast<int64_t>(kv_head) << a.cache.page_shift)) * head_dim;
      }
      *reinterpret_cast<uint4*>(out + low_at) = low[h];
      *reinterpret_cast<uint4*>(out + high_at) = high[h];
    }
  }
}

template <typename T, bool kInterleaved, bool kBias>
void launch_layout(const PagedAppendArgs& a, cudaStream_t stream) {
  // without q_out the query heads of the rows are not read
  const int first_head = a.q_out != nullptr ? 0 : a.query_heads;
  const int heads = a.query_heads + 2 * a.cache.kv_heads - first_head;
  const int units = a.cache.head_dim / 16;
  const int rotated_units = a.rotary_dim / 16;
  // few rows: one a CTA and one head an item, for latency; many: cos, sin and the place lookup are
  // shared by four heads and four rows
  if (a.batch.tokens <= sm_count() * 2) {
    paged_append_kernel<T, kInterleaved, kBias, 1, 1>
        <<<a.batch.tokens, kThreads, 0, stream>>>(a, first_head, units, rotated_units, heads);
  } else {
    paged_append_kernel<T, kInterleaved, kBias, 4, 4>
        <<<(a.batch.tokens + 3) / 4, kThreads, 0, stream>>>(a, first_head, units, rotated_units, (heads + 3) / 4);
  }
}

template <typename T>
void launch_typed(const PagedAppendArgs& a, cudaStream_t stream) {
  if (a.interleaved) {
    a.bias != nullptr ? launch_layout<T, true, true>(a, stream) : launch_layout<T, true, false>(a, stream);
  } else {
    a.bias != nullptr ? launch_layout<T, false, true>(a, stream) : launch_layout<T, false, false>(a, stream);
  }
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs& args, cudaStream_t stream) {
  if (args.batch.tokens <= 0 || args.batch.sequences <= 0) return cudaSuccess;
  args.cache.dtype == kActFp16 ? launch_typed<__half>(args, stream) : launch_typed<__nv_bfloat16>(args, stream);
  return cudaGetLastError();
}

}  // namespace arb
