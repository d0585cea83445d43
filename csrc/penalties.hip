// Penalties, biases and grammar masks on logits (gfx950), x = logits[r, v] in fp32:
//
//   seen token:      x = x > 0 ? x / repetition : x * repetition      (prompt or generated)
//   generated token: x -= frequency * count + presence
//   x += bias[v];    not allowed: x = -inf, whatever x was
//
// A workgroup owns one row and a slice of the vocabulary: it counts the row's history into LDS (an integer per
// vocabulary entry of the slice: the generated count, and a bit for "seen"), then makes one pass over the slice.
// Integer LDS atomics: the result does not depend on their order.
#include "paged.h"

namespace dpa {

namespace {

constexpr int kPenThreads = 512;
constexpr int kPenSlice = 8192;           // vocabulary entries per workgroup
constexpr unsigned kSeen = 0x80000000u;

template <typename T>
__global__ __launch_bounds__(kPenThreads) void penalties_kernel(PenaltyArgs a) {
  __shared__ unsigned cnt[kPenSlice];
  const int row = blockIdx.y, v0 = blockIdx.x * kPenSlice, nv = min(kPenSlice, a.V - v0), tid = threadIdx.x;
  int total = 0;
  if (a.tokens != nullptr) {
    total = a.total_lens != nullptr ? a.total_lens[(long long)row * a.total_stride] : a.L;
    total = min(max(total, 0), a.L);
  }
  if (total > 0) {
    const int prompt = a.prompt_lens != nullptr ? a.prompt_lens[(long long)row * a.prompt_stride] : 0;
    for (int i = tid; i < nv; i += kPenThreads) cnt[i] = 0u;
    __syncthreads();
    for (int j = tid; j < total; j += kPenThreads) {
      const long long at = (long long)row * a.tokens_ld + j;
      const long long tok = a.tokens64 ? ((const long long*)a.tokens)[at] : (long long)((const int*)a.tokens)[at];
      const long long v = tok - v0;
      if (v >= 0 && v < nv) {
        atomicOr(&cnt[v], kSeen);
        if (j >= prompt) atomicAdd(&cnt[v], 1u);
      }
    }
    __syncthreads();
  }
  const float rep = a.repetition != nullptr ? a.repetition[(long long)row * a.repetition_stride] : a.repetition_v;
  const float pres = a.presence != nullptr ? a.presence[(long long)row * a.presence_stride] : a.presence_v;
  const float freq = a.frequency != nullptr ? a.frequency[(long long)row * a.frequency_stride] : a.frequency_v;
  const T* x = (const T*)a.logits + (long long)row * a.ld + v0;
  T* y = (T*)a.out + (long long)row * a.out_ld + v0;
  const float* bias = a.bias != nullptr ? a.bias + (long long)row * a.bias_ld + v0 : nullptr;
  const int* allowed = a.allowed != nullptr ? a.allowed + (long long)row * a.allowed_ld : nullptr;
  for (int i = tid; i < nv; i += kPenThreads) {
    float f = Cvt<T>::ld(x + i);
    if (total > 0) {
      const unsigned c = cnt[i];
      if (c != 0u) {
        f = f > 0.f ? f / rep : f * rep;
        const unsigned n = c & ~kSeen;
        if (n != 0u) f -= freq * (float)n + pres;
      }
    }
    if (bias != nullptr) f += bias[i];
    if (allowed != nullptr && !((allowed[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1)) f = -INFINITY;
    Cvt<T>::st(y + i, f);
  }
}

}  // namespace

void penalize_logits(const PenaltyArgs& a, int num_cus, hipStream_t st) {
  (void)num_cus;
  if (a.R == 0 || a.V == 0) return;
  const dim3 grid((a.V + kPenSlice - 1) / kPenSlice, a.R), block(kPenThreads);
  if (a.type == kTypeBf16) hipLaunchKernelGGL((penalties_kernel<bf16_t>), grid, block, 0, st, a);
  else if (a.type == kTypeHalf) hipLaunchKernelGGL((penalties_kernel<half_t>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((penalties_kernel<float>), grid, block, 0, st, a);
}

}  // namespace dpa
