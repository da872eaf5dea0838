// Rotary positions: cos/sin tables scaled for long contexts, and the rotation of part of a head in
// the half or the interleaved layout (contracts in include/attnrank_b200.h).
//
// Table: the angle p f is formed in quarter turns, p (4 f / 2 pi), in fp64 (an fp32 product loses all
// digits of the fraction near 2^24 turns and is off by 1e-3 rad at 1e4) and split there into its
// nearest whole number n of quarters and the remainder u in [-1/2, 1/2]; sin and cos of pi/2 u are
// polynomials in fp32, n's low bits swap them and give their signs. A thread keeps its column's
// frequency and walks down the positions, so a value costs five fp64 and about twenty other operations.
// Their issue bounds it, not the 8 bytes a value, which stay in L2: 128K positions x 32 pairs (33.5 MB) take
// 10.2 us a call, half of the measured copy, with 73% of the issue slots used, the integer and logic pipe 55%
// busy and fp64 11% (12.9 us with sincospi of the fp32 remainder in place of the polynomials).
//
// Rotation: y_a = a c - b s, y_b = b c + a s, one read and one write of each 16-bit value: HBM bounds
// it (16K tokens x 32 heads x 128, half of each head: 45.3 to 46.6 us a call, 0.89 to 0.91 of the measured copy).
#include <algorithm>

#include "common.cuh"
#include "layer_kernels.h"
#include "paged.h"

namespace arb {
namespace {

constexpr int kThreads = 256;
constexpr int kTableUnroll = 2;  // positions a thread computes before it stores

// (sin, cos) of `quarter` quarter turns. The polynomials have the least largest error on [-1/2, 1/2] (Remez
// exchange): 1.2e-9 for sin, 5.4e-11 for cos; 3.0e-8 and 6.7e-9 with the coefficients rounded to fp32, 1.1e-7 and
// 7.5e-8 with the roundings of u and of each step, checked at 44 million points. That is 1.5 times the error of
// an fp64 value rounded once, chosen for the time above.
__device__ __forceinline__ void sincos_quarters(double quarter, float& s, float& c) {
  const double shifted = quarter + 6755399441055744.0;  // 1.5 x 2^52: the sum's low bits hold the nearest integer
  const int n = __double2loint(shifted);
  const float u = static_cast<float>(quarter - (shifted - 6755399441055744.0));
  const float z = u * u;
  float sine = fmaf(-0.004592289216816425f, z, 0.07967590540647507f);
  sine = fmaf(sine, z, -0.6459629535675049f);
  sine = fmaf(sine, z, 1.570796251296997f) * u;
  float cosine = fmaf(0.0009040216682478786f, z, -0.02086028829216957f);
  cosine = fmaf(cosine, z, 0.25366923213005066f);
  cosine = fmaf(cosine, z, -1.2337005138397217f);
  cosine = fmaf(cosine, z, 1.0f);
  s = (n & 1) ? cosine : sine;
  c = (n & 1) ? sine : cosine;
  s = __int_as_float(__float_as_int(s) ^ ((n & 2) << 30));
  c = __int_as_float(__float_as_int(c) ^ (((n + 1) & 2) << 30));
}

// A block takes `rows` positions at a time, thread t column t % half of row t / half; blocks take turns.
__global__ void __launch_bounds__(kThreads) rope_table_scaled_kernel(const __grid_constant__ TableTurns turns, int half,
                                                                     int rows, float multiplier, int positions,
                                                                     float* __restrict__ cos_table,
                                                                     float* __restrict__ sin_table) {
  const int row = threadIdx.x / half;
  const int column = threadIdx.x - row * half;
  if (row >= rows) return;
  const double frequency = 4.0 * turns.value[column];
  const int step = gridDim.x * rows;
  int64_t at = static_cast<int64_t>(blockIdx.x) * rows * half + threadIdx.x;
  for (int position = blockIdx.x * rows + row; position < positions; position += kTableUnroll * step) {
    float s[kTableUnroll], c[kTableUnroll];
#pragma unroll
    for (int i = 0; i < kTableUnroll; ++i) {
      sincos_quarters((static_cast<double>(position) + static_cast<double>(i * step)) * frequency, s[i], c[i]);
    }
#pragma unroll
    for (int i = 0; i < kTableUnroll; ++i) {
      if (positions - position > i * step) {
        __stcs(cos_table + at, c[i] * multiplier);
        __stcs(sin_table + at, s[i] * multiplier);
      }
      at += static_cast<int64_t>(step) * half;
    }
  }
}

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  return static_cast<float>(v);
}

// Vector form: an item is one token, kHeads heads and one unit of 16 values of each: eight rotation
// pairs, or sixteen values behind the rotated part.
template <typename T, bool kInterleaved, int kHeads>
__global__ void __launch_bounds__(kThreads) rotary_positions_kernel(const RotaryArgs a, int units, int rotated_units,
                                                                    int groups, int64_t items) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (item >= items) return;
  const int unit = static_cast<int>(item % units);
  const int64_t rest = item / units;
  const int group = static_cast<int>(rest % groups);
  const int token = static_cast<int>(rest / groups);
  const int position = __ldg(a.positions + token);
  if (position < 0 || position >= a.table_positions) {
    report_status(a.status, kStatusPositionOutOfRange);
    return;
  }
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
  const bool high_in = high_at < a.head_dim;
  const int first = group * kHeads;
  const T* x = static_cast<const T*>(a.x) + token * a.x_token_stride;
  T* out = static_cast<T*>(a.out) + token * a.out_token_stride;
  uint4 low[kHeads], high[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (first + h < a.heads) {
      const T* row = x + (first + h) * a.x_head_stride;
      low[h] = *reinterpret_cast<const uint4*>(row + low_at);
      if (high_in) high[h] = *reinterpret_cast<const uint4*>(row + high_at);
    }
  }
  float c[8], s[8];
  if (rotated) {
    const int64_t at = static_cast<int64_t>(position) * (a.rotary_dim >> 1) + unit * 8;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 c4 = __ldg(reinterpret_cast<const float4*>(a.cos_table + at + i));
      const float4 s4 = __ldg(reinterpret_cast<const float4*>(a.sin_table + at + i));
      c[i] = c4.x, c[i + 1] = c4.y, c[i + 2] = c4.z, c[i + 3] = c4.w;
      s[i] = s4.x, s[i + 1] = s4.y, s[i + 2] = s4.z, s[i + 3] = s4.w;
    }
    if (a.inverse) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = -s[i];
    }
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (first + h >= a.heads) break;
    if (rotated) rotate16<T, kInterleaved>(low[h], high[h], c, s);
    T* row = out + (first + h) * a.out_head_stride;
    *reinterpret_cast<uint4*>(row + low_at) = low[h];
    if (high_in) *reinterpret_cast<uint4*>(row + high_at) = high[h];
  }
}

// Form for sizes, strides or addresses that do not hold 16-byte accesses: an item is one token,
// kHeads heads and one rotation pair, or two values behind the rotated part. Its accesses of 2 bytes bound
// it, a warp's being 64 neighbouring bytes in the half layout and every other value, twice, interleaved: 16K
// tokens x 32 heads x 128 take 102 us with 66 values rotated (half) and 88 us with 126 (interleaved), against
// 49 us in the vector form with 64 or 128 and a floor of 41 us; cold cache, timed alone.
template <typename T, bool kInterleaved, int kHeads>
__global__ void __launch_bounds__(kThreads) rotary_positions_pairs_kernel(const RotaryArgs a, int units,
                                                                          int rotated_units, int groups,
                                                                          int64_t items) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (item >= items) return;
  const int unit = static_cast<int>(item % units);
  const int64_t rest = item / units;
  const int group = static_cast<int>(rest % groups);
  const int token = static_cast<int>(rest / groups);
  const int position = __ldg(a.positions + token);
  if (position < 0 || position >= a.table_positions) {
    report_status(a.status, kStatusPositionOutOfRange);
    return;
  }
  const bool rotated = unit < rotated_units;
  int low_at, high_at;
  if (!rotated) {
    low_at = a.rotary_dim + (unit - rotated_units) * 2;
    high_at = low_at + 1;
  } else if (kInterleaved) {
    low_at = unit * 2;
    high_at = low_at + 1;
  } else {
    low_at = unit;
    high_at = rotated_units + unit;
  }
  const bool high_in = high_at < a.head_dim;
  const int first = group * kHeads;
  const T* x = static_cast<const T*>(a.x) + token * a.x_token_stride;
  T* out = static_cast<T*>(a.out) + token * a.out_token_stride;
  T low[kHeads], high[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (first + h < a.heads) {
      const T* row = x + (first + h) * a.x_head_stride;
      low[h] = row[low_at];
      if (high_in) high[h] = row[high_at];
    }
  }
  float c = 1.0f, s = 0.0f;
  if (rotated) {
    const int64_t at = static_cast<int64_t>(position) * rotated_units + unit;
    c = __ldg(a.cos_table + at);
    s = __ldg(a.sin_table + at);
    if (a.inverse) s = -s;
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (first + h >= a.heads) break;
    T* row = out + (first + h) * a.out_head_stride;
    if (rotated) {
      const float l = to_float(low[h]);
      const float r = to_float(high[h]);
      low[h] = static_cast<T>(l * c - r * s);
      high[h] = static_cast<T>(r * c + l * s);
    }
    row[low_at] = low[h];
    if (high_in) row[high_at] = high[h];
  }
}

template <typename T, bool kInterleaved>
void launch_layout(const RotaryArgs& a, cudaStream_t stream) {
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out) |
                              reinterpret_cast<uintptr_t>(a.cos_table) | reinterpret_cast<uintptr_t>(a.sin_table);
  const int64_t strides = a.x_token_stride | a.x_head_stride | a.out_token_stride | a.out_head_stride;
  const bool vectors = addresses % 16 == 0 && strides % 8 == 0 && a.head_dim % 8 == 0 && a.rotary_dim % 16 == 0;
  const bool in_place = a.out == a.x;  // the values behind the rotated part are there already
  const int width = vectors ? 16 : 2;
  const int rotated_units = a.rotary_dim / width;
  const int units = in_place ? rotated_units : rotated_units + (a.head_dim - a.rotary_dim + width - 1) / width;
  auto run = [&](auto kernel, int heads_per_item) {
    const int groups = (a.heads + heads_per_item - 1) / heads_per_item;
    const int64_t per_token = static_cast<int64_t>(groups) * units;
    const int step = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(a.tokens, (int64_t{1} << 30) / per_token)));
    for (int64_t begin = 0; begin < a.tokens; begin += step) {  // one launch but for batches beyond 2^30 items
      RotaryArgs part = a;
      part.tokens = static_cast<int>(std::min<int64_t>(step, a.tokens - begin));
      part.x = static_cast<const T*>(a.x) + begin * a.x_token_stride;
      part.out = static_cast<T*>(a.out) + begin * a.out_token_stride;
      part.positions = a.positions + begin;
      const int64_t items = part.tokens * per_token;
      kernel<<<static_cast<unsigned>((items + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
          part, units, rotated_units, groups, items);
    }
  };
  // one head an item while that does not fill the GPU, four (one read of cos and sin for them) above
  const bool few = static_cast<int64_t>(a.tokens) * a.heads * units <= static_cast<int64_t>(sm_count()) * kThreads * 4;
  if (vectors) {
    few ? run(rotary_positions_kernel<T, kInterleaved, 1>, 1) : run(rotary_positions_kernel<T, kInterleaved, 4>, 4);
  } else {
    few ? run(rotary_positions_pairs_kernel<T, kInterleaved, 1>, 1)
        : run(rotary_positions_pairs_kernel<T, kInterleaved, 4>, 4);
  }
}

}  // namespace

cudaError_t launch_rope_table_scaled(const TableTurns& turns, int half, float multiplier, int positions,
                                     float* cos_table, float* sin_table, cudaStream_t stream) {
  if (positions <= 0) return cudaSuccess;
  const int rows = kThreads / half;
  const int64_t blocks = (static_cast<int64_t>(positions) + rows - 1) / rows;
  const int grid = static_cast<int>(std::min<int64_t>(blocks, static_cast<int64_t>(sm_count()) * 8));
  rope_table_scaled_kernel<<<grid, kThreads, 0, stream>>>(turns, half, rows, multiplier, positions, cos_table, sin_table);
  return cudaGetLastError();
}

cudaError_t launch_rotary_positions(const RotaryArgs& args, cudaStream_t stream) {
  if (args.tokens <= 0 || args.heads <= 0) return cudaSuccess;
  if (args.dtype == kActFp16) {
    args.interleaved ? launch_layout<__half, true>(args, stream) : launch_layout<__half, false>(args, stream);
  } else {
    args.interleaved ? launch_layout<__nv_bfloat16, true>(args, stream)
                     : launch_layout<__nv_bfloat16, false>(args, stream);
  }
  return cudaGetLastError();
}

}  // namespace arb
