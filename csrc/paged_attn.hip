// Causal attention of the newest tokens of every request over its pages (gfx950). Row i of request r sits at position
// pos = kv[r] - n[r] + i - cu[r] (n[r] = cu[r + 1] - cu[r]) and attends keys max(0, pos - window + 1) .. pos:
//
//   o[i, h] = sum_j softmax_j(scale q[i, h] . K[r, j, g]) V[r, j, g],   g = h / (nh / nkv)
//
// A key whose table entry names no page of the pool is left out; a row that sees no key gives zeros.
//
// Any type, width (<= 256) and stride: one wave per (row, head). Lane = key for the scores of 64 keys at a time, then
// lane = feature for the values, probabilities by broadcast; running maximum, sum and output in fp32.
#include "paged.h"

namespace dpa {

namespace {

constexpr int kGenWaves = 4;
constexpr int kGenWidth = 256;

// Request of row i: the last r with cu[r] <= i (cu does not decrease).
__device__ __forceinline__ int request_of(const int* cu, int R, int i) {
  int lo = 0, hi = R;   // cu[lo] <= i < cu[hi] once the ends are checked by the caller
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(kGenWaves * 64) void paged_attn_rows_kernel(PagedAttnArgs a) {
  __shared__ float q_s[kGenWaves][kGenWidth];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long id = (long long)blockIdx.x * kGenWaves + wave;
  if (id >= (long long)a.N * a.nh) return;     // whole waves; no workgroup barrier below
  const int i = (int)(id / a.nh), h = (int)(id % a.nh), g = h / (a.nh / a.nkv);
  T* o = (T*)a.o + (long long)i * a.o_ts + (long long)h * a.o_hs;
  const int nd = (a.width + 63) / 64;
  if (a.R == 0 || i < a.cu_q[0] || i >= a.cu_q[a.R]) {
    if (a.zero_rest)
      for (int d = lane; d < a.width; d += 64) Cvt<T>::st(o + d, 0.f);
    return;
  }
  const int r = request_of(a.cu_q, a.R, i);
  const int start = a.cu_q[r], n = a.cu_q[r + 1] - start;
  const int pos = a.kv_lens[r] - n + i - start;
  const long long cap = (long long)a.M * a.page;
  const int last = (int)min((long long)pos, cap - 1);
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const T* q = (const T*)a.q + (long long)i * a.q_ts + (long long)h * a.q_hs;
  for (int d = lane; d < a.width; d += 64) q_s[wave][d] = Cvt<T>::ld(q + d) * a.scale;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

  const int* row_table = a.table + (long long)r * a.table_ld;
  float m = -INFINITY, l = 0.f, acc[kGenWidth / 64];
#pragma unroll
  for (int j = 0; j < kGenWidth / 64; ++j) acc[j] = 0.f;
  for (int k0 = lo; k0 <= last; k0 += 64) {
    const int key = k0 + lane;
    int pg = -1, row = 0;
    if (key <= last) {
      const int col = fast_div(key, a.by_page);
      pg = row_table[col];
      row = key - col * a.page;
      if (pg < 0 || pg >= a.pages) pg = -1;
    }
    float s = -INFINITY;
    if (pg >= 0) {
      const T* k = (const T*)a.k + pg * a.k_ps + row * a.k_rs + g * a.k_hs;
      s = 0.f;
      for (int d = 0; d < a.width; ++d) s += q_s[wave][d] * Cvt<T>::ld(k + d);
    }
    const float mx = wave_max(s);
    const float mn = fmaxf(m, mx);
    const float base = mn == -INFINITY ? 0.f : mn;      // nothing seen yet: every exponential below is exp(-inf)
    const float p = pg >= 0 ? __expf(s - base) : 0.f;
    const float alpha = __expf(m - base);
    l = l * alpha + wave_sum(p);
    m = mn;
#pragma unroll
    for (int j = 0; j < kGenWidth / 64; ++j) acc[j] *= alpha;
    for (int t = 0; t < 64; ++t) {
      const int tp = __shfl(pg, t, 64), tr = __shfl(row, t, 64);
      const float pt = __shfl(p, t, 64);
      if (tp < 0) continue;
      const T* v = (const T*)a.v + tp * a.v_ps + tr * a.v_rs + g * a.v_hs;
#pragma unroll
      for (int j = 0; j < kGenWidth / 64; ++j)
        if (j < nd && lane + 64 * j < a.width) acc[j] += pt * Cvt<T>::ld(v + lane + 64 * j);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < kGenWidth / 64; ++j)
    if (j < nd && lane + 64 * j < a.width) Cvt<T>::st(o + lane + 64 * j, l == 0.f ? 0.f : acc[j] * inv);
}

}  // namespace

void paged_attn(const PagedAttnArgs& a, hipStream_t st) {
  if (a.N == 0 || a.nh == 0) return;
  const long long waves = (long long)a.N * a.nh;
  const dim3 grid((unsigned)((waves + kGenWaves - 1) / kGenWaves)), block(kGenWaves * 64);
  if (a.type == kTypeBf16) hipLaunchKernelGGL((paged_attn_rows_kernel<bf16_t>), grid, block, 0, st, a);
  else if (a.type == kTypeHalf) hipLaunchKernelGGL((paged_attn_rows_kernel<half_t>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged_attn_rows_kernel<float>), grid, block, 0, st, a);
}

}  // namespace dpa
