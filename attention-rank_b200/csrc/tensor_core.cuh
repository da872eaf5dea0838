// tcgen05 helpers of the paged chunk attention: descriptors of 128-byte-swizzled operands, MMA issue,
// TMEM loads and stores, packed fp32 pairs.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace arb {
namespace tc {

// K-major 128B-swizzled operand: 128-byte rows, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t address) {
  return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// MN-major 128B-swizzled operand (V as B of P.V): each 128-byte row holds 64 consecutive N (head dim)
// values of one K (key); the 64-wide N halves are `half_bytes` apart, 8-key groups 1024 bytes.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t address, uint32_t half_bytes) {
  return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (static_cast<uint64_t>(half_bytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// kind::f16 instruction descriptor, fp32 accumulator, M = 128, N = n; format 0 = fp16, 1 = bf16 (A and
// B always of the same format); A K-major, B K-major or MN-major.
constexpr uint32_t idesc(uint32_t format, bool b_mn_major, uint32_t n) {
  return (1u << 4) | (format << 7) | (format << 10) | (b_mn_major ? (1u << 16) : 0u) | ((n >> 3) << 17) |
         ((128u >> 4) << 24);
}
// True in one lane of the converged warp. A warp that walks its loop as a whole and issues through
// this keeps descriptors in uniform registers; under `if (lane == 0)` each MMA moved its operands there
// one by one.
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(elected));
  return elected != 0;
}
// D (TMEM) = A (shared) B (shared) (+ D)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
// D (TMEM) = A (TMEM) B (shared) (+ D)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t address, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(address));
}
__device__ __forceinline__ void tmem_st32(uint32_t address, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(address), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Packed fp32 pairs (f32x2 arithmetic): one instruction does two values' FMA or add.
__device__ __forceinline__ unsigned long long pack_f32x2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(unsigned long long v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b,
                                                        unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// max(a, b, c) in one instruction; NaN if any of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^t of kPairs pairs on the FMA pipe, for finite t below 127: 2^t = 2^n 2^f, n the nearest integer
// (found by adding 1.5 x 2^23, whose sum keeps n in its low bits), 2^f on [-1/2, 1/2] by the polynomial
// of degree 5 with the least largest relative error (7.5e-8; 2.2e-7 with the fp32 roundings, checked at
// 2 million points), n added to the exponent. Below 2^-125 it stays there. Step by step over all pairs,
// so that a step's latency is hidden behind the others'.
template <int kPairs>
__device__ __forceinline__ void exp2_fma(const unsigned long long (&t)[kPairs], float (&p)[2 * kPairs]) {
  unsigned long long clamped[kPairs], shifted[kPairs], f[kPairs], y[kPairs];
  const auto both = [](float v) { return pack_f32x2(v, v); };
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    float t0, t1;
    unpack_f32x2(t[i], t0, t1);
    clamped[i] = pack_f32x2(fmaxf(t0, -125.0f), fmaxf(t1, -125.0f));
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) shifted[i] = add_f32x2(clamped[i], both(12582912.0f));
#pragma unroll
  for (int i = 0; i < kPairs; ++i) f[i] = add_f32x2(shifted[i], both(-12582912.0f));
#pragma unroll
  for (int i = 0; i < kPairs; ++i) f[i] = fma_f32x2(f[i], both(-1.0f), clamped[i]);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) y[i] = fma_f32x2(both(0.0013276472454890609f), f[i], both(0.009675541892647743f));
#pragma unroll
  for (int i = 0; i < kPairs; ++i) y[i] = fma_f32x2(y[i], f[i], both(0.05550713092088699f));
#pragma unroll
  for (int i = 0; i < kPairs; ++i) y[i] = fma_f32x2(y[i], f[i], both(0.24022120237350464f));
#pragma unroll
  for (int i = 0; i < kPairs; ++i) y[i] = fma_f32x2(y[i], f[i], both(0.6931469440460205f));
#pragma unroll
  for (int i = 0; i < kPairs; ++i) y[i] = fma_f32x2(y[i], f[i], both(1.0000001192092896f));
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    float s0, s1, y0, y1;
    unpack_f32x2(shifted[i], s0, s1);
    unpack_f32x2(y[i], y0, y1);
    p[2 * i] = __uint_as_float(__float_as_uint(y0) + (__float_as_uint(s0) << 23));
    p[2 * i + 1] = __uint_as_float(__float_as_uint(y1) + (__float_as_uint(s1) << 23));
  }
}
// A whole 32-byte sector in one store (two 16-byte stores each write half of one).
__device__ __forceinline__ void store_sector(void* to, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

}  // namespace tc
}  // namespace arb
