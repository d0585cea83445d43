// Shared pieces of the paged-cache kernels (csrc/paged_plan.hip, paged_append.hip, paged_attn.hip) and csrc/penalties.hip.
#pragma once
#include "common.h"
#include "kernels.h"

namespace dpa {

typedef _Float16 half_t;

template <> struct Cvt<half_t> {
  static __device__ __forceinline__ float ld(const half_t* p) { return (float)*p; }
  static __device__ __forceinline__ void st(half_t* p, float v) { *p = (half_t)v; }   // round to nearest even
};

__device__ __forceinline__ void load8(const half_t* p, float (&o)[8]) {
  typedef __attribute__((ext_vector_type(8))) _Float16 half8;
  const half8 v = *reinterpret_cast<const half8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (float)v[i];
}
__device__ __forceinline__ void store8(half_t* p, const float (&o)[8]) {
  typedef __attribute__((ext_vector_type(8))) _Float16 half8;
  half8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (half_t)o[i];
  *reinterpret_cast<half8*>(p) = v;
}

// n / d for 0 <= n < 2^31 and a divisor known on the host: q = (n + hi32(n * mul)) >> shift with
// shift = ceil(log2 d), mul = floor(2^32 (2^shift - d) / d) + 1 (the round-up method of division by invariant integers;
// the sum stays below 2^32 because hi32(n * mul) <= n).
__device__ __forceinline__ int fast_div(int n, const FastDiv& f) {
  return (int)((__umulhi((unsigned)n, f.mul) + (unsigned)n) >> f.shift);
}

}  // namespace dpa
