// Results that workgroups of one launch hand over: relaxed 64-bit accesses at agent scope, past the L2 of an XCD.  The writer waits for
// its stores (s_waitcnt vmcnt(0)) before it tells the reader; a release fence would write that L2 back.
#pragma once
#include "common.h"

namespace xot {

__device__ __forceinline__ void agent_store2(float* p, float a, float b) {
  const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_store4(float* p, const f32x4& v) {
  agent_store2(p, v[0], v[1]);
  agent_store2(p + 2, v[2], v[3]);
}
__device__ __forceinline__ f32x2_t agent_load2(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return {__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}
__device__ __forceinline__ f32x4 agent_load4(const float* p) {
  const f32x2_t a = agent_load2(p), b = agent_load2(p + 2);
  return {a[0], a[1], b[0], b[1]};
}

}  // namespace xot
