// Attention of new tokens over a paged KV cache (contract in include/attnrank_b200.h). For a row
// (token at position p, query head h):
//   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = scale log2(e) q . k_j,  m = max_j x_j,
//   lse = m + log2 sum_j 2^(x_j - m),
// over the visible positions, in one pass with the running maximum and sum.
//
// One warp per row: lane l holds values l * D / 32 .. of q and of the accumulator, a score is a warp
// sum, and positions the row does not see are never read.
#include <cmath>

#include "common.cuh"
#include "layer_kernels.h"
#include "paged.h"

namespace arb {
namespace {

constexpr int kThreads = 128;

template <typename T, int kDim>
__device__ __forceinline__ void load_lane(const T* row, float (&v)[kDim / 32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kDim / 64; ++i) {
    const auto pair = reinterpret_cast<const typename Pair<T>::type*>(row)[lane * (kDim / 64) + i];
    const float2 f = Pair<T>::to_float2(pair);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads) paged_attention_rows_kernel(const PagedAttentionArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int token = static_cast<int>(row / a.query_heads);
  const int head = static_cast<int>(row - static_cast<int64_t>(token) * a.query_heads);
  if (token >= a.batch.tokens) return;
  const int s = paged_sequence_of(a.batch, token);
  if (s < 0) return;
  const PagedSequence seq = paged_sequence(a.batch, s, a.status);
  const int index = token - seq.q_begin;
  if (index < 0 || index >= seq.q_len) return;
  const int position = seq.kv_len - seq.q_len + index;
  const int kv_head = head / (a.query_heads / a.cache.kv_heads);
  const int first = a.sliding_window > 0 ? max(0, position - a.sliding_window + 1) : 0;
  constexpr int kValues = kDim / 32;
  float q[kValues], o[kValues];
  load_lane<T, kDim>(static_cast<const T*>(a.q) + token * a.q_stride + head * kDim, q);
#pragma unroll
  for (int i = 0; i < kValues; ++i) o[i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  const int page_size = 1 << a.cache.page_shift;
  for (int begin = first; begin <= position;) {
    const int page = paged_page(a.cache, a.batch, s, begin >> a.cache.page_shift, a.status);
    const int end = min(position + 1, (begin | (page_size - 1)) + 1);
    const int64_t base = ((static_cast<int64_t>(page) * a.cache.kv_heads + kv_head) << a.cache.page_shift);
    for (int j = begin; j < end; ++j) {
      const int64_t at = (base + (j & (page_size - 1))) * kDim;
      float k[kValues], v[kValues];
      load_lane<T, kDim>(static_cast<const T*>(a.cache.k_pages) + at, k);
      load_lane<T, kDim>(static_cast<const T*>(a.cache.v_pages) + at, v);
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < kValues; ++i) dot = fmaf(q[i], k[i], dot);
      const float x = warp_sum(dot) * a.scale_log2;
      const float top = fmaxf(m, x);
      const float keep = exp2f(m - top);  // 0 on the first key
      const float p = exp2f(x - top);
      l = l * keep + p;
#pragma unroll
      for (int i = 0; i < kValues; ++i) o[i] = o[i] * keep + p * v[i];
      m = top;
    }
    begin = end;
  }
  const float inverse = position >= first ? 1.0f / l : 0.0f;
  T* out = static_cast<T*>(a.out) + token * a.out_stride + head * kDim;
#pragma unroll
  for (int i = 0; i < kDim / 64; ++i) {
    reinterpret_cast<typename Pair<T>::type*>(out)[lane * (kDim / 64) + i] =
        Pair<T>::from_floats(o[2 * i] * inverse, o[2 * i + 1] * inverse);
  }
  if (lane == 0 && a.lse != nullptr) {
    a.lse[static_cast<int64_t>(token) * a.query_heads + head] = position >= first ? m + log2f(l) : -INFINITY;
  }
}

}  // namespace

int64_t paged_attention_workspace(const PagedCache&, const PagedBatch&, int) { return 0; }

cudaError_t launch_paged_attention(const PagedAttentionArgs& a, cudaStream_t stream) {
  if (a.batch.tokens <= 0 || a.batch.sequences <= 0) return cudaSuccess;
  const int64_t rows = static_cast<int64_t>(a.batch.tokens) * a.query_heads;
  const int64_t grid = (rows + kThreads / 32 - 1) / (kThreads / 32);
  auto run = [&](auto kernel) { kernel<<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a); };
  if (a.cache.dtype == kActFp16) {
    a.cache.head_dim == 128 ? run(paged_attention_rows_kernel<__half, 128>) : run(paged_attention_rows_kernel<__half, 64>);
  } else {
    a.cache.head_dim == 128 ? run(paged_attention_rows_kernel<__nv_bfloat16, 128>)
                            : run(paged_attention_rows_kernel<__nv_bfloat16, 64>);
  }
  return cudaGetLastError();
}

}  // namespace arb
