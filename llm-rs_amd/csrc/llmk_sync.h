// llmk_sync.h — how the operators around the sampling kernels pass words
// between waves and between workgroups.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llmk {

// A barrier for LDS alone: requests to memory stay on their way across it
// (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Words that one workgroup hands to another, or that two of them write one after
// the other, within a launch: at agent scope, past the XCDs' own caches, ordered
// by waiting for the stores (wait_stores).  A fence per workgroup instead, which
// writes its XCD's whole L2 back, took 131 us instead of 29 for 256 rows of 8
// workgroups each (llmk_logprobs, 151936 f32 logits a row).
__device__ __forceinline__ void put_agent(uint32_t* p, uint32_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t get_agent(const uint32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace llmk
