// mbarrier and TMA helpers of the paged attention kernels, and the tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "common.cuh"

namespace arb {
namespace async {

constexpr uint32_t kSpinLimit = 1u << 26;                // hard backstop on polls per wait
constexpr uint64_t kWaitLimitNs = 500ull * 1000 * 1000;  // a wait gives up after 0.5 s

__device__ __forceinline__ uint32_t smem_u32(const void* pointer) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(pointer));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The arrival of the lanes with `elected` not 0, without a branch.
__device__ __forceinline__ void mbar_arrive_if(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}"
      ::"r"(bar), "r"(elected)
      : "memory");
}
__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t phase) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(phase)
      : "memory");
  return done != 0;
}
// Bounded wait for the completion of phase `phase` (parity): gives up after kWaitLimitNs (or
// kSpinLimit polls), or earlier once *abort is set by another thread of the CTA.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t phase, const volatile int* abort) {
  uint64_t start = 0;
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try(bar, phase)) return true;
    if ((i & 1023) == 1023) {
      if (abort != nullptr && *abort) return false;
      const uint64_t now = global_ns();
      if (start == 0) {
        start = now;
      } else if (now - start > kWaitLimitNs) {
        return false;
      }
    }
  }
  return false;
}
// The same with the loop in a function of its own, for a kernel that waits at many places with few live
// registers: the copies of the loop crowd the instruction cache (830 -> 800 us for two 4K chunks in the
// chunk attention; in the few-row attention, whose accumulators are live, the call spills: 193 -> 202).
static __device__ __noinline__ bool mbar_wait_loop(uint32_t bar, uint32_t phase, const volatile int* abort) {
  return mbar_wait(bar, phase, abort);
}
// The wait of a role that carries on when it gives up: it reports the timeout and sets *abort, after
// which every such wait returns at once and the rest of the work runs through on what is there.
static __device__ __noinline__ void mbar_wait_or_abort(uint32_t bar, uint32_t phase, volatile int* abort, int* status) {
  if (*abort) return;
  if (mbar_wait(bar, phase, abort)) return;
  report_status(status, kStatusWaitTimeout);
  *abort = 1;
}
__device__ __forceinline__ bool mbar_wait_called(uint32_t bar, uint32_t phase, const volatile int* abort) {
  return mbar_try(bar, phase) || mbar_wait_loop(bar, phase, abort);
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// Programmatic dependent launch: wait for the preceding kernel's completion and writes; let the next
// kernel of the stream be scheduled.
__device__ __forceinline__ void wait_for_producer() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void release_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// 2^x with the SFU's ex2 instruction, results below 2^-126 flushed to zero.
__device__ __forceinline__ float ex2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace async

// Launches with programmatic stream serialization: the kernel may start while the one before it on the
// stream ends, and every thread of it calls wait_for_producer() before it reads or writes memory.
template <typename... Parameters, typename... Arguments>
cudaError_t launch_overlapped(void (*kernel)(Parameters...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream,
                              Arguments... arguments) {
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, arguments...);
}

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* pointer = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &pointer, cudaEnableDefault, &result) == cudaSuccess &&
        result == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(pointer);
    }
  });
  return fn;
}

}  // namespace arb
