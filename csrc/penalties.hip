// Penalties, biases and grammar masks on logits (gfx950), x = logits[r, v] in fp32:
//
//   seen token:      x = x > 0 ? x / repetition : x * repetition      (prompt or generated)
//   generated token: x -= frequency * count + presence
//   x += bias[v];    not allowed: x = -inf, whatever x was
//
// A workgroup owns one row and a slice of the vocabulary: it counts the row's history into LDS, one counter per entry
// of the slice (the generated count, and a top bit for "in the prompt"), then makes one pass over the slice. Integer
// LDS atomics: the result does not depend on their order. Bound by the logits' bytes at serving batches and by
// latency at a few rows, so the slice is what fills the card: a whole row's worth of it costs one pass over the
// history per slice, a short one spreads a few rows over many CUs. Counters have 16 bits while the history cannot
// overflow the 15 of the count. Measured: one row of 50304 bf16 4.0 us (7.3 us a call from Python); 256 rows fp32 with
// bias, mask and 2000-4000 tokens of history 33 us, 5.0 TB/s (8192 entries to a slice with 32-bit counters and single
// elements: 69 us).
#include <algorithm>

#include "paged.h"

namespace dpa {

namespace {

constexpr int kPenThreads = 512;
constexpr int kPenLds = 52 * 1024;        // counters of a workgroup: three workgroups on a CU
constexpr int kPenMin = 1024;             // entries below which a slice is not worth a workgroup
constexpr int kPenUnroll = 4;

__device__ __forceinline__ float penalized(float f, unsigned c, unsigned seen_bit, float rep, float freq, float pres) {
  if (c != 0u) {
    f = f > 0.f ? f / rep : f * rep;
    const unsigned n = c & (seen_bit - 1u);
    if (n != 0u) f -= freq * (float)n + pres;
  }
  return f;
}

// C: counter (uint16_t or unsigned); VEC: 8 = rows allow 16-byte accesses, 1 = single elements
template <typename T, typename C, int VEC>
__global__ __launch_bounds__(kPenThreads) void penalties_kernel(PenaltyArgs a, int slice) {
  constexpr unsigned kSeen = 1u << (sizeof(C) * 8 - 1);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  C* cnt = reinterpret_cast<C*>(smem);
  const int row = blockIdx.y, v0 = blockIdx.x * slice, nv = min(slice, a.V - v0), tid = threadIdx.x;
  int total = 0;
  if (a.tokens != nullptr) {
    total = a.total_lens != nullptr ? a.total_lens[(long long)row * a.total_stride] : a.L;
    total = min(max(total, 0), a.L);
  }
  const int prompt = a.prompt_lens != nullptr ? a.prompt_lens[(long long)row * a.prompt_stride] : 0;
  const float rep = a.repetition != nullptr ? a.repetition[(long long)row * a.repetition_stride] : a.repetition_v;
  const float pres = a.presence != nullptr ? a.presence[(long long)row * a.presence_stride] : a.presence_v;
  const float freq = a.frequency != nullptr ? a.frequency[(long long)row * a.frequency_stride] : a.frequency_v;
  if (total > 0) {
    for (int i = tid; i * 16 < nv * (int)sizeof(C); i += kPenThreads) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    auto count = [&](long long tok, int j) {
      const long long v = tok - v0;
      if (v < 0 || v >= nv) return;
      const unsigned what = j >= prompt ? 1u : kSeen;
      if (sizeof(C) == 4) {
        if (what == 1u) atomicAdd(reinterpret_cast<unsigned*>(smem) + v, 1u);
        else atomicOr(reinterpret_cast<unsigned*>(smem) + v, kSeen);
      } else {
        unsigned* w = reinterpret_cast<unsigned*>(smem) + (v >> 1);
        const int sh = 16 * (int)(v & 1);
        if (what == 1u) atomicAdd(w, 1u << sh);
        else atomicOr(w, kSeen << sh);
      }
    };
    for (int j0 = tid; j0 < total; j0 += kPenThreads * kPenUnroll) {
      long long tok[kPenUnroll];
#pragma unroll
      for (int u = 0; u < kPenUnroll; ++u) {
        const long long at = (long long)row * a.tokens_ld + min(j0 + u * kPenThreads, total - 1);
        tok[u] = a.tokens64 ? ((const long long*)a.tokens)[at] : (long long)((const int*)a.tokens)[at];
      }
#pragma unroll
      for (int u = 0; u < kPenUnroll; ++u)
        if (j0 + u * kPenThreads < total) count(tok[u], j0 + u * kPenThreads);
    }
    __syncthreads();
  }
  const T* x = (const T*)a.logits + (long long)row * a.ld + v0;
  T* y = (T*)a.out + (long long)row * a.out_ld + v0;
  const float* bias = a.bias != nullptr ? a.bias + (long long)row * a.bias_ld + v0 : nullptr;
  const int* allowed = a.allowed != nullptr ? a.allowed + (long long)row * a.allowed_ld + (v0 >> 5) : nullptr;   // v0 % 32 == 0
  const int n = nv / VEC;      // VEC == 8: V % 8 == 0
  for (int i0 = tid; i0 < n; i0 += kPenThreads * kPenUnroll) {
    float f[kPenUnroll][VEC], b[kPenUnroll][VEC];
    int word[kPenUnroll];
#pragma unroll
    for (int u = 0; u < kPenUnroll; ++u) {
      const int i = min(i0 + u * kPenThreads, n - 1);
      if constexpr (VEC == 8) {
        load8(x + i * 8, f[u]);
        if (bias != nullptr) load8(bias + i * 8, b[u]);
      } else {
        f[u][0] = Cvt<T>::ld(x + i);
        if (bias != nullptr) b[u][0] = bias[i];
      }
      word[u] = allowed != nullptr ? allowed[(i * VEC) >> 5] : -1;
    }
#pragma unroll
    for (int u = 0; u < kPenUnroll; ++u) {
      const int i = i0 + u * kPenThreads;
      if (i >= n) break;
      if (total > 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[u][e] = penalized(f[u][e], cnt[i * VEC + e], kSeen, rep, freq, pres);
      }
      if (bias != nullptr) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[u][e] += b[u][e];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (!((word[u] >> ((i * VEC + e) & 31)) & 1)) f[u][e] = -INFINITY;
      if constexpr (VEC == 8) store8(y + i * 8, f[u]);
      else Cvt<T>::st(y + i, f[u][0]);
    }
  }
}

template <typename T, typename C>
void launch(const PenaltyArgs& a, int slice, bool wide, hipStream_t st) {
  const dim3 grid((a.V + slice - 1) / slice, a.R), block(kPenThreads);
  const size_t lds = a.tokens != nullptr ? (size_t)slice * sizeof(C) : 0;
  if (wide) hipLaunchKernelGGL((penalties_kernel<T, C, 8>), grid, block, lds, st, a, slice);
  else hipLaunchKernelGGL((penalties_kernel<T, C, 1>), grid, block, lds, st, a, slice);
}
template <typename T>
void launch(const PenaltyArgs& a, int num_cus, hipStream_t st) {
  const bool narrow = a.L < (1 << 15);
  const int most = narrow ? kPenLds / 2 : kPenLds / 4;
  const int wgs = std::max((2 * num_cus + a.R - 1) / a.R, 1);       // per row, for two on every CU
  int slice = std::min(std::max((a.V + wgs - 1) / wgs, kPenMin), most);
  slice = (slice + 31) / 32 * 32;
  const int es = 16 / (int)sizeof(T);
  const bool wide = a.V % 8 == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 &&
                    (a.R == 1 || (a.ld % es == 0 && a.out_ld % es == 0)) &&
                    (a.bias == nullptr || (reinterpret_cast<uintptr_t>(a.bias) % 16 == 0 && (a.R == 1 || a.bias_ld % 4 == 0)));
  if (narrow) launch<T, uint16_t>(a, slice, wide, st);
  else launch<T, unsigned>(a, slice, wide, st);
}

}  // namespace

void penalize_logits(const PenaltyArgs& a, int num_cus, hipStream_t st) {
  if (a.R == 0 || a.V == 0) return;
  if (a.type == kTypeBf16) launch<bf16_t>(a, num_cus, st);
  else if (a.type == kTypeHalf) launch<half_t>(a, num_cus, st);
  else launch<float>(a, num_cus, st);
}

}  // namespace dpa
