// Causal attention of the newest tokens of every request over its pages (gfx950). Row i of request r sits at position
// pos = kv[r] - n[r] + i - cu[r] (n[r] = cu[r + 1] - cu[r]) and attends keys max(0, pos - window + 1) .. pos:
//
//   o[i, h] = sum_j softmax_j(scale q[i, h] . K[r, j, g]) V[r, j, g],   g = h / (nh / nkv)
//
// A key whose table entry names no page of the pool is left out; a row that sees no key gives zeros.
//
// Any type, width (<= 256) and stride: one wave per (row, head). Lane = key for the scores of 64 keys at a time, then
// lane = feature for the values, probabilities by broadcast; running maximum, sum and output in fp32.
#include <algorithm>
#include <cmath>

#include "mfma_tiles.h"
#include "paged.h"
#include "paged_items.h"

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
  const long long id = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * kGenWaves + wave;
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


// ---------------------------------------------------------------------------------------------------------
// bf16 / fp16, widths up to 128 in whole 16-byte pieces: matrix instructions.
//
// The G = nh / nkv query heads of a KV head share its keys, so a request's rows are (token, head of the group) pairs
// packed per KV head; K and V are read once per tile of rows, not once per head. An item is (request, row tile, KV
// head, piece of the keys):
//   few rows (at most 32 packed, a decode step): the four waves of a workgroup take 32-key subtiles in turn, each
//     through its own part of LDS without any workgroup barrier, and are merged at the end. Bound by K / V bytes.
//   chunks: 128 packed rows, 32 per wave, over 64-key tiles that the waves share (two stages). Bound by products.
// Both use the same step: S^T = K Q^T (v_mfma 32x32x16, lane = row, keys along the accumulator), running maximum and
// sum per lane, O^T += V^T P^T with V read transposed from LDS.
//
// Lengths live on the device, so every workgroup derives the list of items from them (one pass over the requests:
// R <= 256 is one load per lane or thread; more go through one more kernel). Few rows alone (paged_attn_few_kernel) take
// equal shares of all 128-key steps, one round of workgroups whatever the lengths. Chunks (paged_attn_kernel, few rows
// among them) take items; their keys are cut into pieces when there are fewer items than `target`. What is cut leaves
// (O, reference, sum) in the workspace and a second kernel joins it, in the order of the keys: a result does not
// depend on which workgroup ran when. The second kernel costs 4 - 6 us of every call.
//
// Measured (large copy on the same card 4.9 TB/s, plain reads 6.2, a large bf16 product 1.48 PF/s):
//   64 requests x 2000-8000 keys, 32 / 8 heads of 128, bf16      215 us   5.9 TB/s: the bytes
//   2 requests x 33 K-131 K keys, same heads, fp16               106 us   5.7 TB/s
//   8 requests x 250-1000 keys, 12 heads of 64, bf16              17 us   four dependent trips to memory (lengths, table,
//                                                                         keys, join) on a quarter-empty card
//   8 prompts of 1000-3000 rows on 500-2000 cached, 32 / 8 x 128  640 - 680 us  0.81 - 0.86 PF/s: the matrix pipes are
//                                                                         busy 38 % of the time, the CUs hold waves 95 %
//   8 prompts of 2048 rows, 16 heads of 64                       112 - 116 us  0.6 PF/s
// The first form of a page's addresses that fits is taken (64 x 8000 keys of 128): whole runs of 16 rows in a page 230 us,
// of 4 (pages of 20) 240, an address per lane (pages of 18) 260.
//
// Two things the loops live from, both found in the compiler's waits: nothing in them may spill (a reload is a
// vector-memory wait, which waits for the transfers in flight: 737 -> 1232 us on the prompts), so what is rare is done
// elsewhere (exact_rows); and no register that an ordinary load fills may have its first use in them (load_row).
//
// The score's reference point mb (log2 units) does not follow every new maximum. Few rows move it when a subtile's
// maximum passes mb + kBias + 8, chunks when 16 keys sum to more than kSumMax: p <= 2^8 for bf16 either way, 2^14 (few
// rows) or 2^15 (chunks) for fp16. kBias = 6 for fp16 keeps small probabilities out of its subnormal range (one of 2^-20
// still has all its bits). The output is divided by the sum at the end, so 2^8 |v| times the number of keys has to stay
// below fp32's 3.4e38: bf16 values up to 1e30 with 2^20 keys and a reference as far off as it gets.
// Scores are scaled in fp32 after the product: q keeps its bits. A negative scale negates q, which is exact.
// ---------------------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
using namespace paged;
constexpr int kThreads = 256;

template <typename T> struct Frag;
template <> struct Frag<bf16_t> {
  static constexpr int kBias = 0;
  static constexpr unsigned kExp = 0x7f807f80u, kExpOne = 0x00800080u;     // both halves' exponents, and their last bits
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfrag, a), __builtin_bit_cast(bfrag, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float lower(unsigned x) { return __uint_as_float(x << 16); }
  static __device__ __forceinline__ float upper(unsigned x) { return __uint_as_float(x & 0xffff0000u); }
};
template <> struct Frag<half_t> {
  static constexpr int kBias = 6;
  static constexpr unsigned kExp = 0x7c007c00u, kExpOne = 0x04000400u;
  typedef __attribute__((ext_vector_type(8))) _Float16 half8;
  typedef __attribute__((ext_vector_type(2))) _Float16 half2_t;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned pack(float lo, float hi) {
    half2_t v;
    v[0] = (half_t)lo;     // round to nearest even
    v[1] = (half_t)hi;
    return __builtin_bit_cast(unsigned, v);
  }
  static __device__ __forceinline__ float lower(unsigned x) { return (float)__builtin_bit_cast(half2_t, x)[0]; }
  static __device__ __forceinline__ float upper(unsigned x) { return (float)__builtin_bit_cast(half2_t, x)[1]; }
};

struct FastArgs {
  float c;             // |scale| log2 e
  bool negate;         // scale < 0
  int G;               // query heads per KV head
  FastDiv by_group;
  int target;          // items wanted on the card
  bool stream;         // the pools are larger than the memory-side cache
  int max_slots, slot_rows;
  float* part;         // [max_slots][slot_rows][W] unnormalised outputs of pieces
  float* ml;           // [max_slots][slot_rows][2] reference, sum
  int* meta;           // [max_slots][8]
  int* header;         // [0] = slots in use, [1], [2] = keys per piece (R > kWaveRequests), [3] = cu_q decreases
  int* prefix;         // R > kWaveRequests: [3][R + 1] first items (few rows: steps), slots and second items before each request
};

// 256 zero bytes: what rows that no query may see, and pages that do not exist, read as
__device__ __attribute__((aligned(256))) const unsigned zero_row[64] = {};

// Inclusive prefix sum over the wave by register moves between lanes (shifts inside rows of 16, then row broadcasts).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
__device__ __forceinline__ float wave_total(float x) {
  auto dpp = [](float v, auto ctrl, auto rows) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
#define DPA_STEP(ctrl, rows) x += dpp(x, std::integral_constant<int, ctrl>(), std::integral_constant<int, rows>())
  DPA_STEP(0x111, 0xf);
  DPA_STEP(0x112, 0xf);
  DPA_STEP(0x114, 0xf);
  DPA_STEP(0x118, 0xf);
  DPA_STEP(0x142, 0xa);
  DPA_STEP(0x143, 0xc);
#undef DPA_STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Many requests, whose prefixes lie in memory: the last r with prefix[r] <= x < prefix[R], 64 of them at a time.
__device__ __forceinline__ int find_prefix(const int* prefix, int R, int x, int lane) {
  int lo = 0, n = R;
  if (x >= prefix[R]) return -1;
  while (n > 1) {
    const int per = (n + 63) >> 6, at = lo + lane * per;
    const unsigned long long below = __ballot(lane * per < n && prefix[at] <= x);
    if (below == 0ull) return -1;
    const int src = 63 - __builtin_clzll(below);
    n = min(per, n - src * per);
    lo += src * per;
  }
  return lo;
}

struct Item {
  int r, j, slot, np;      // request, number inside it, slot of its output, pieces of its keys; r < 0: none
};
// Item `id`, found by one wave; every wave of the grid comes to the same list. The list goes over the requests twice,
// first the last two thirds of each one's tiles, which see most, then the others: the card runs out of work on short
// items while those that run together still share a request's keys (8 x 2048 rows of 16 heads of 64 123 -> 112 us, mixed
// batch 36.5 -> 35.4, no difference on the 16k prompts; halves 115 us, three quarters 119).
__device__ __forceinline__ Item find_item(const PagedAttnArgs& a, const FastArgs& f, int id, int lane) {
  Item it;
  it.r = -1;
  if (a.R <= kWaveRequests) {
    constexpr int PER = kWaveRequests / 64;      // consecutive requests per lane
    Request q[PER];
    float cost = 0.f;
    bool back = false;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      q[u].tiles = 0;
      const int per = (a.R + 63) >> 6, r = lane * per + u;
      if (u < per && r < a.R) {
        q[u] = request(a, f.G, r);
        cost += request_cost(q[u]);
        back |= q[u].back;
      }
    }
    const int any_back = __any(back);
    if (id == 0) f.header[3] = any_back;
    if (any_back) return it;
    const PieceSize size = piece_size(wave_total(cost), a.nkv, f.target);
    int items[PER], ahead[PER], slots[PER], n1 = 0, n2 = 0, ns = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      items[u] = ahead[u] = slots[u] = 0;
      if (q[u].tiles > 0) {
        const int np = pieces(q[u], size);
        ahead[u] = first_items(q[u], np, a.nkv);
        items[u] = second_items(q[u], np, a.nkv);
        slots[u] = np > 1 ? ahead[u] + items[u] : 0;
      }
      n1 += ahead[u];
      n2 += items[u];
      ns += slots[u];
    }
    const int p1 = wave_scan(n1), p2 = wave_scan(n2), ps = wave_scan(ns);
    if (id == 0 && lane == 63) f.header[0] = min(ps, f.max_slots);
    const int all1 = __builtin_amdgcn_readlane(p1, 63);
    const bool second = id >= all1;
    const int pi = second ? p2 : p1, ni = second ? n2 : n1;
    id -= second ? all1 : 0;
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (!second) {
        items[u] = ahead[u];
        ahead[u] = 0;
      }
    const unsigned long long here = __ballot(id >= pi - ni && id < pi);
    if (here == 0ull) return it;
    const int src = __builtin_ctzll(here);
    int first = pi - ni, slot = ps - ns, u = 0;
    // the request of that lane
#pragma unroll
    for (int v = 0; v + 1 < PER; ++v)
      if (u == v && id >= first + items[v]) {
        first += items[v];
        slot += slots[v];
        u = v + 1;
      }
    int np = 1;
#pragma unroll
    for (int v = 0; v < PER; ++v)
      if (u == v && q[v].tiles > 0) {
        np = pieces(q[v], size);
        first -= ahead[v];
      }
    it.r = src * ((a.R + 63) >> 6) + __builtin_amdgcn_readlane(u, src);
    it.j = id - __builtin_amdgcn_readlane(first, src);
    it.slot = __builtin_amdgcn_readlane(slot, src) + it.j;
    it.np = __builtin_amdgcn_readlane(np, src);
    return it;
  }
  if (f.header[3] != 0) return it;
  const int* const second = f.prefix + 2 * (a.R + 1);
  const int all1 = f.prefix[a.R];
  const int lo = id < all1 ? find_prefix(f.prefix, a.R, id, lane) : find_prefix(second, a.R, id - all1, lane);
  if (lo < 0) return it;
  it.r = lo;
  it.j = id < all1 ? id - f.prefix[lo] : f.prefix[lo + 1] - f.prefix[lo] + id - all1 - second[lo];
  it.slot = f.prefix[a.R + 1 + lo] + it.j;
  const Request q = request(a, f.G, lo);
  PieceSize size;
  size.few = f.header[1];
  size.chunk = f.header[2];
  it.np = pieces(q, size);
  return it;
}

// ---- few rows only: equal shares of all steps ----
// A (request, 32 packed rows, KV head) is a run of 128-key steps (one at least); the runs lie one after another, and workgroup i of `eff`
// takes steps [i * per, (i + 1) * per) of them all, whichever runs they fall into: contexts of any mix of lengths load
// the card evenly in one round. At most its first and its last run are cut. One step is worth a workgroup of its own (8 x
// 1k keys: 17.2 us; two at least: 19.7, four: 20.9, eight, uncut: 31.7).

struct Runs {        // the requests of the batch in LDS (R <= kWaveRequests)
  int before[kWaveRequests + 1];       // steps before each
  int start[kWaveRequests], rows[kWaveRequests], shift[kWaveRequests];
  int red[kThreads / 64];
  int back[kThreads / 64];
};
static_assert(kWaveRequests == kThreads, "one request per thread");
// Steps of all runs, none if cu_q decreases; leaves `runs` filled for every thread.
__device__ __forceinline__ int list_runs(const PagedAttnArgs& a, const FastArgs& f, Runs& runs) {
  if (a.R > kWaveRequests) return f.header[3] != 0 ? 0 : f.prefix[a.R];
  const int tid = threadIdx.x;
  int steps = 0;
  bool back = false;
  if (tid < a.R) {
    const Request q = request(a, f.G, tid);
    steps = run_steps(q) * run_count(q, a.nkv);
    back = q.back;
    runs.start[tid] = q.start;
    runs.rows[tid] = q.rows;
    runs.shift[tid] = q.shift;
  }
  int incl = wave_scan(steps);
  if (a.R > 64) {
    if ((tid & 63) == 63) runs.red[tid >> 6] = incl;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64 - 1; ++w)
      if (w < (tid >> 6)) incl += runs.red[w];
  }
  if (tid < a.R) runs.before[tid + 1] = incl;
  if (tid == 0) runs.before[0] = 0;
  const int any_back = __any(back);
  if ((tid & 63) == 0) runs.back[tid >> 6] = any_back;
  __syncthreads();
  const int bad = runs.back[0] | runs.back[1] | runs.back[2] | runs.back[3];
  if (blockIdx.x == 0 && tid == 0) f.header[3] = bad;
  return __builtin_amdgcn_readfirstlane(bad != 0 ? 0 : runs.before[a.R]);
}
// The request of step `at`, and the number of its first step; r < 0: there is none.
__device__ __forceinline__ int find_run(const PagedAttnArgs& a, const FastArgs& f, const Runs& runs, int at, int& first, Request& q) {
  const int lane = threadIdx.x & 63;
  if (a.R > kWaveRequests) {
    const int r = find_prefix(f.prefix, a.R, at, lane);
    if (r < 0) return -1;
    first = __builtin_amdgcn_readfirstlane(f.prefix[r]);
    q = request(a, f.G, r);
    return r;
  }
  int below = 0;
  for (int u = 0; u < a.R; u += 64) below += __popcll(__ballot(u + lane < a.R && runs.before[u + lane] <= at));
  const int r = below - 1;
  if (r < 0) return -1;
  first = __builtin_amdgcn_readfirstlane(runs.before[r]);
  q.start = __builtin_amdgcn_readfirstlane(runs.start[r]);
  q.rows = __builtin_amdgcn_readfirstlane(runs.rows[r]);
  q.shift = __builtin_amdgcn_readfirstlane(runs.shift[r]);
  q.n = fast_div(q.rows, f.by_group);
  key_range(a, q);
  return r;
}

// The prefixes for many requests: one workgroup.
template <bool CHUNKS>
__global__ __launch_bounds__(1024) void paged_attn_items_kernel(PagedAttnArgs a, FastArgs f) {
  __shared__ float red_f[16];
  __shared__ int red[3][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float cost = 0.f;
  bool back = false;
  for (int r = tid; r < a.R; r += 1024) {
    const Request q = request(a, f.G, r);
    if (CHUNKS) cost += request_cost(q);
    back |= q.back;
  }
  if (CHUNKS) cost = block_sum(cost, red_f);
  back = __syncthreads_or(back);
  if (tid == 0) f.header[3] = back;
  if (back) return;
  PieceSize size{};
  if constexpr (CHUNKS) size = piece_size(cost, a.nkv, f.target);
  // scans of the first items (few rows: steps), and for chunks of the second items and the slots
  constexpr int NS = CHUNKS ? 3 : 1;
  int* const out[3] = {f.prefix, f.prefix + 2 * (a.R + 1), f.prefix + a.R + 1};
  int base[NS] = {};
  for (int r0 = 0; r0 < a.R; r0 += 1024) {
    const int r = r0 + tid;
    int n[NS] = {};
    if (r < a.R) {
      const Request q = request(a, f.G, r);
      if constexpr (CHUNKS) {
        const int np = pieces(q, size);
        n[0] = first_items(q, np, a.nkv);
        n[1] = second_items(q, np, a.nkv);
        n[2] = np > 1 ? n[0] + n[1] : 0;
      } else {
        n[0] = run_steps(q) * run_count(q, a.nkv);
      }
    }
    int p[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      p[i] = wave_scan(n[i]);
      if (lane == 63) red[i][wave] = p[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      int total = 0;
      for (int w = 0; w < 16; ++w) {
        if (w == wave) p[i] += total;
        total += red[i][w];
      }
      if (r < a.R) out[i][r] = base[i] + p[i] - n[i];
      base[i] += total;
    }
    __syncthreads();
  }
  if (tid == 0) {
    out[0][a.R] = base[0];
    if constexpr (CHUNKS) {
      out[1][a.R] = base[1];
      f.header[0] = min(base[2], f.max_slots);
      f.header[1] = size.few;
      f.header[2] = size.chunk;
    }
  }
}

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_dma_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// 1 KiB global -> LDS, one 16-byte piece per lane: from a scalar base plus the lane's offset, or from the lane's address.
template <bool NT>
__device__ __forceinline__ void dma_uniform(unsigned long long base, unsigned voff, unsigned dst) {
  if (NT)
    asm volatile(
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %2 nt"
        :
        : "v"(voff), "s"(dst), "s"(base)
        : "memory", "m0");
  else
    asm volatile(
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %2"
        :
        : "v"(voff), "s"(dst), "s"(base)
        : "memory", "m0");
}
__device__ __forceinline__ void dma_lane(unsigned long long addr, unsigned dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(addr), "s"(dst)
      : "memory", "m0");
}

// NP pieces (1 KiB transfers of RPP rows of W columns) of pages -> LDS. RUN: rows that are known to lie in one page, since
// the page size is a multiple of it and the row fills the tile: the page number and the address of a run come from
// scalar registers, its pieces are lane offsets. RUN = 0: nothing is known, every lane looks its row up (any page size,
// rows narrower than the tile).
template <int W, int NP, int RUN>
struct PageRows {
  static constexpr int CPR = W / 8, RPP = 64 / CPR, PER = RUN > 0 ? RUN / RPP : 1, NR = NP / PER;    // pieces per run, runs
  static constexpr int VAR = W == 128 ? 4 : 2;      // the swizzle of a piece repeats after VAR pieces
  static constexpr int OFF = PER > VAR ? PER : VAR;
  const PagedAttnArgs* a;
  const int* table;       // the request's row
  unsigned long long kb, vb;
  int klo, khi, lane;
  bool gone;              // a page of the rows fetched last does not exist
  unsigned kv_off[2][OFF];
  int pg[RUN > 0 ? NR : NP];

  __device__ __forceinline__ void init(const PagedAttnArgs& args, const int* t, int g, int lo, int hi, int lane_) {
    a = &args;
    table = t;
    klo = lo;
    khi = hi;
    gone = false;
    lane = lane_;
    kb = (unsigned long long)args.k + 2ull * (unsigned long long)(g * args.k_hs);
    vb = (unsigned long long)args.v + 2ull * (unsigned long long)(g * args.v_hs);
#pragma unroll
    for (int v = 0; v < OFF; ++v) {
      const int row = v * RPP + lane / CPR;
      const unsigned col = 16u * swz<W>(row, lane % CPR);
      const int in_run = (v % PER) * RPP + lane / CPR;
      kv_off[0][v] = (unsigned)in_run * (unsigned)(2 * args.k_rs) + col;
      kv_off[1][v] = (unsigned)in_run * (unsigned)(2 * args.v_rs) + col;
    }
  }
  // Every row exists and somebody may see it: all lanes transfer, and a transfer is one instruction per piece.
  __device__ __forceinline__ bool whole(int ks0) const { return RUN > 0 && !gone && ks0 >= klo && ks0 + NP * RPP <= khi; }
  // page numbers of the rows [ks0, ks0 + NP * RPP), for the issue() of those rows; known() waits for them
  __device__ __forceinline__ void fetch(int ks0) {
    if constexpr (RUN > 0) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int col = fast_div(min(ks0 + i * RUN, khi - 1), a->by_page);
        typedef const __attribute__((address_space(4))) int* scalar_ptr;
        pg[i] = *(scalar_ptr)(unsigned long long)(table + __builtin_amdgcn_readfirstlane(col));
      }
    } else {
#pragma unroll
      for (int pc = 0; pc < NP; ++pc) {
        const int key = ks0 + pc * RPP + lane / CPR;
        pg[pc] = key >= klo && key < khi ? table[fast_div(key, a->by_page)] : -1;
      }
    }
  }
  __device__ __forceinline__ void known(int ks0) {
    bool bad = false;
    if constexpr (RUN > 0) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int r0 = ks0 + i * RUN;
        bad |= r0 < khi && r0 + RUN > klo && (unsigned)pg[i] >= (unsigned)a->pages;
      }
    } else {
#pragma unroll
      for (int pc = 0; pc < NP; ++pc) {
        const int key = ks0 + pc * RPP + lane / CPR;
        bad |= key >= klo && key < khi && (unsigned)pg[pc] >= (unsigned)a->pages;
      }
      bad = __any(bad);
    }
    gone = bad;
  }
  // `stream` (few rows over pools past the memory-side cache: every byte is read once): without a place in the caches.
  // Rows that no query may see, and rows of missing pages, become zeros.
  template <bool V>
  __device__ __forceinline__ void issue(int ks0, unsigned lds, bool stream = false) const {
    const unsigned long long base = V ? vb : kb;
    const unsigned ps = 2u * (unsigned)(V ? a->v_ps : a->k_ps), rs = 2u * (unsigned)(V ? a->v_rs : a->k_rs);
    if constexpr (RUN > 0) {
      unsigned long long from[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int key = min(ks0 + i * RUN, khi - 1);
        const unsigned row = __builtin_amdgcn_readfirstlane(key - fast_div(key, a->by_page) * a->page) & ~(RUN - 1);
        const unsigned p = __builtin_amdgcn_readfirstlane(pg[i]);
        from[i] = base + (unsigned long long)p * ps + row * rs;
      }
      if (whole(ks0)) {
        if (stream) {
#pragma unroll
          for (int pc = 0; pc < NP; ++pc) dma_uniform<true>(from[pc / PER], kv_off[V][pc % OFF], lds + pc * 1024);
        } else {
#pragma unroll
          for (int pc = 0; pc < NP; ++pc) dma_uniform<false>(from[pc / PER], kv_off[V][pc % OFF], lds + pc * 1024);
        }
        return;
      }
#pragma unroll
      for (int pc = 0; pc < NP; ++pc) {
        const int key = ks0 + pc * RPP + lane / CPR;
        if ((unsigned)pg[pc / PER] < (unsigned)a->pages && key >= klo && key < khi)
          dma_uniform<false>(from[pc / PER], kv_off[V][pc % OFF], lds + pc * 1024);    // (lanes that are off leave their place alone)
        else
          *(__attribute__((address_space(3))) u32x4*)(size_t)(lds + pc * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
      }
    } else {
#pragma unroll
      for (int pc = 0; pc < NP; ++pc) {
        const int row = pc * RPP + lane / CPR, key = ks0 + row;
        const int ch = swz<W>(row, lane % CPR), p = pg[pc];
        unsigned long long addr = (unsigned long long)zero_row + 16u * ch;
        const int col = fast_div(max(key, 0), a->by_page);
        if ((unsigned)p < (unsigned)a->pages && ch * 8 < a->width)      // (-1: nobody sees the row)
          addr = base + (unsigned long long)(unsigned)p * ps + (unsigned)(key - col * a->page) * rs + 16u * ch;
        dma_lane(addr, lds + pc * 1024);
      }
    }
  }
};

// One lane's row: bounds of the keys it sees, reference, sum (of its half of the keys) and the output tile.
template <int W>
struct RowState {
  int lo, hi;
  float mb, l;
  f32x16 o[W / 32];
  __device__ __forceinline__ void clear() {
    mb = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < W / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  }
};

__device__ __forceinline__ void swap_halves(float& x, float& y) {
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 0" : "+v"(x), "+v"(y));
}
__device__ __forceinline__ float max_halves(float x) {
  float u = x, v = x;
  swap_halves(u, v);
  return fmaxf(u, v);
}
__device__ __forceinline__ float sum_halves(float x) {
  float u = x, v = x;
  swap_halves(u, v);
  return u + v;
}

// Whether any of the wave's values is not finite.
template <typename T, int W>
__device__ __forceinline__ bool not_finite(const u32x4 (&vf)[2][W / 32]) {
  unsigned bad = 0u;
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
    for (int dt = 0; dt < W / 32; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) bad |= (vf[s2][dt][j] & Frag<T>::kExp) + Frag<T>::kExpOne;   // carries into the sign
  return __any((bad & 0x80008000u) != 0u);
}

// A 32-key subtile: keys [ks0, ks0 + 32) in the LDS tiles kt, vt. mask: some of them are hidden from some row of the wave;
// returns whether one of their values is not finite then (exact_rows).
template <typename T, int W, class AfterK, class BeforeV, class AfterV>
__device__ __forceinline__ bool subtile(const char* kt, const char* vt, int ks0, bool mask, float c, const u32x4 (&qf)[W / 16],
                                        RowState<W>& st, int lane, AfterK after_k, BeforeV before_v, AfterV after_v) {
  typedef Frag<T> F;
  constexpr int NK = W / 16, ND = W / 32;
  const int r = lane & 31, hh = lane >> 5;
  u32x4 kf[NK];
#pragma unroll
  for (int ks = 0; ks < NK; ++ks) kf[ks] = __builtin_bit_cast(u32x4, row_frag<W>(kt, r, ks, hh));
  after_k();
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
  for (int ks = 0; ks < NK; ++ks) s = F::mfma(kf[ks], qf[ks], s);
  const int lo_rel = st.lo - ks0, hi_rel = st.hi - ks0;
  if (mask) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = acc_row(i, hh);
      if (key < lo_rel || key > hi_rel) s[i] = -INFINITY;
    }
  }
  float mx = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
  mx = max_halves(mx) * c;
  const bool move = mx > st.mb + (float)(F::kBias + 8);      // the first key a row sees moves it from -inf
  if (__any(move)) {
    const float to = mx - (float)F::kBias;
    const float alpha = move ? __builtin_amdgcn_exp2f(st.mb - to) : 1.f;
    st.mb = move ? to : st.mb;
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[dt][i] *= alpha;
  }
  before_v();
  u32x4 vf[2][ND];
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) vf[s2][dt] = __builtin_bit_cast(u32x4, tr_frag<W>(vt, 0, s2, dt, lane));
  const float base = st.mb == -INFINITY ? 0.f : st.mb;       // no key seen yet: every s is -inf
  float rs = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -base));
    rs += s[i];
  }
  st.l += rs;
  after_v();
  bool rare = false;
  if (mask) rare = not_finite<T, W>(vf);
  // A probability goes in as two 16-bit parts, the second what the first leaves out: 16 bits of it for bf16, 22 for fp16. The
  // products hide behind the bytes (64 x 8k 213 -> 216.5 us, 2 x 128k 105 -> 106, 8 x 1k 17.15 -> 17.35).
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) {
    u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = s[8 * s2 + 2 * j], y = s[8 * s2 + 2 * j + 1];
      hi[j] = F::pack(x, y);
      lo[j] = F::pack(x - F::lower(hi[j]), y - F::upper(hi[j]));
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
      st.o[dt] = F::mfma(vf[s2][dt], hi, st.o[dt]);
      st.o[dt] = F::mfma(vf[s2][dt], lo, st.o[dt]);
    }
  }
  return rare;
}

// A 32-key subtile of a chunk, from key ks0 on. No maximum is taken as a rule: the probabilities come from the
// reference as it is, and what they sum to says whether it still serves (fp32 sums and the 16-bit operand keep their
// relative precision whatever the magnitude; kSumMax keeps fp16 finite). If it does not, or a row has none yet, the
// scores are computed again and the reference moves to their maximum. (Two subtiles taken together: 668 instead of 653
// us on the 16k prompts, fewer registers to schedule with.)
// Behind the score products a wave goes before the others of its SIMD: one is then in its softmax and value products
// while another waits for its keys, where equals would do both at the same time (16k prompts 665 -> 640 us, mixed batch
// 35.2 -> 33.7; from the key reads on 648, for the products alone 664, for the softmax alone 664).
template <typename T, int W>
__device__ __forceinline__ bool chunk_tile(const char* kt, const char* vt, int ks0, bool mask, float c, const u32x4 (&qf)[W / 16],
                                           RowState<W>& st, int lane) {
  typedef Frag<T> F;
  constexpr int NK = W / 16, ND = W / 32;
  constexpr float kSumMax = F::kBias ? 32768.f : 256.f;
  const int r = lane & 31, hh = lane >> 5;
  f32x16 s;
  auto scores = [&]() {
    u32x4 kf[NK];
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) kf[ks] = __builtin_bit_cast(u32x4, row_frag<W>(kt, r, ks, hh));
    __builtin_amdgcn_sched_barrier(0);     // all fragments requested before the first product
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) s = F::mfma(kf[ks], qf[ks], s);
    __builtin_amdgcn_s_setprio(1);
    if (mask) {
      const int lo_rel = st.lo - ks0 - 4 * hh, hi_rel = st.hi - ks0 - 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = acc_row(i, 0);
        if (key < lo_rel || key > hi_rel) s[i] = -INFINITY;
      }
    }
  };
  auto weights = [&]() {
    const float base = st.mb == -INFINITY ? 0.f : st.mb;      // a row that sees nothing yet: every s is -inf
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -base));
      sum[i & 1] += s[i];
    }
    return sum[0] + sum[1];
  };
  scores();
  float rs = weights();
  if (!__all(rs <= kSumMax && (st.mb != -INFINITY || st.hi < 0))) {
    scores();
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    const float to = max_halves(mx) * c - (float)F::kBias;
    const bool move = to > st.mb;
    const float alpha = move ? __builtin_amdgcn_exp2f(st.mb - to) : 1.f;
    st.mb = move ? to : st.mb;
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[dt][i] *= alpha;
    rs = weights();
  }
  st.l += rs;
  u32x4 vf[2][ND];
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) vf[s2][dt] = __builtin_bit_cast(u32x4, tr_frag<W>(vt, 0, s2, dt, lane));
  __builtin_amdgcn_sched_barrier(0);
  bool rare = false;
  if (mask) rare = not_finite<T, W>(vf);
  // Here a probability is rounded to the type, as the matrix instruction takes it: 2^-8 of itself for bf16, averaged over
  // the keys (0.0023 instead of 0.0017 of the result's norm, whose own rounding is the 0.0017). In two parts, as few rows
  // have it, the products cost 16k prompts 660 -> 845 us.
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) {
    u32x4 pb;
#pragma unroll
    for (int j = 0; j < 4; ++j) pb[j] = F::pack(s[8 * s2 + 2 * j], s[8 * s2 + 2 * j + 1]);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) st.o[dt] = F::mfma(vf[s2][dt], pb, st.o[dt]);
  }
  __builtin_amdgcn_s_setprio(0);
  return rare;
}

// fp32 output tile [32 rows][W] of a wave in LDS; 16-byte pieces XORed with the row against bank conflicts.
template <int W>
__device__ __forceinline__ float* o_piece(char* tile, int row, int piece) {
  return reinterpret_cast<float*>(tile + row * (W * 4) + 16 * (piece ^ (row & (W / 4 - 1))));
}

// A tile of packed rows of one request and KV head.
struct Tile {
  int start, shift, rows, rows0, nrows, g;
  int p_first, p_last, klo, khi, cap;      // positions of its first and last row, keys that any of them sees
  const int* table;
};
__device__ __forceinline__ Tile make_tile(const PagedAttnArgs& a, const FastArgs& f, const Request& q, int r, int g, int rows0,
                                          int most) {
  Tile t;
  t.start = q.start;
  t.shift = q.shift;
  t.rows = q.rows;
  t.rows0 = rows0;
  t.nrows = min(most, q.rows - rows0);
  t.g = g;
  t.p_first = q.start + fast_div(rows0, f.by_group) + q.shift;
  t.p_last = q.start + fast_div(rows0 + t.nrows - 1, f.by_group) + q.shift;
  t.cap = a.M * a.page;
  t.khi = max(min(t.p_last + 1, t.cap), 0);
  t.klo = min(a.window > 0 ? max(t.p_first - a.window + 1, 0) : 0, t.khi);
  t.table = a.table + (long long)r * a.table_ld;
  return t;
}
// Packed row i of the tile's request: row of the batch and head.
__device__ __forceinline__ long long row_offset(const FastArgs& f, const Tile& t, int i, long long ts, long long hs) {
  const int tk = fast_div(i, f.by_group);
  return (long long)(t.start + tk) * ts + (long long)(t.g * f.G + i - tk * f.G) * hs;
}
// The lane's row (a packed row, or none): queries as the second operand of the score product, bounds of its keys.
template <int W>
__device__ __forceinline__ void load_row(const PagedAttnArgs& a, const FastArgs& f, const Tile& t, int row, bool valid, int hh,
                                         u32x4 (&qf)[W / 16], RowState<W>& st) {
  st.clear();
  const int pos = t.start + fast_div(valid ? row : 0, f.by_group) + t.shift;
  st.hi = valid ? min(pos, t.cap - 1) : -1;
  st.lo = a.window > 0 ? pos - a.window + 1 : 0;
  const uint16_t* qp = (const uint16_t*)a.q + (valid ? row_offset(f, t, row, a.q_ts, a.q_hs) : 0);
#pragma unroll
  for (int ks = 0; ks < W / 16; ++ks) {
    const int d = ks * 16 + hh * 8;
    qf[ks] = u32x4{0u, 0u, 0u, 0u};
    if (valid && d < a.width) qf[ks] = *reinterpret_cast<const u32x4*>(qp + d);
  }
  if (f.negate) {
#pragma unroll
    for (int ks = 0; ks < W / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[ks][e] ^= 0x80008000u;
  }
  // Have them here: their first use is inside the caller's loop, where the compiler's wait for them would, in every
  // round, wait for the transfers of the next tile as well.
#pragma unroll
  for (int ks = 0; ks < W / 16; ++ks) asm volatile("" : "+v"(qf[ks]));
}
// The rows of a tile over keys [k0, k1) one by one, key by key: what a row does not see takes no part, whatever it holds.
// For tiles with a missing page, or with a value that is not finite in a subtile that some row sees only in part, where a
// product would carry 0 * inf into that row. Kept out of the common loops, whose registers it would spill. qs: LDS.
template <typename T, int W>
__device__ __forceinline__ void exact_rows(const PagedAttnArgs& a, const FastArgs& f, const Tile& t, int k0, int k1, int slot, float* qs) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float c = f.negate ? -f.c : f.c;
  float* const q_s = qs + wave * W;
  for (int rr = wave; rr < t.nrows; rr += kThreads / 64) {
    const int row = t.rows0 + rr;
    const T* q = (const T*)a.q + row_offset(f, t, row, a.q_ts, a.q_hs);
    const int pos = t.start + fast_div(row, f.by_group) + t.shift;
    const int lo = max(k0, a.window > 0 ? max(pos - a.window + 1, 0) : 0), last = min(min(pos, t.cap - 1), k1 - 1);
    for (int d = lane; d < W; d += 64) q_s[d] = d < a.width ? Cvt<T>::ld(q + d) : 0.f;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    float m = -INFINITY, l = 0.f, acc[W / 64];
#pragma unroll
    for (int j = 0; j < W / 64; ++j) acc[j] = 0.f;
    for (int key0 = lo; key0 <= last; key0 += 64) {
      const int key = key0 + lane;
      int pg = -1, in = 0;
      if (key <= last) {
        const int col = fast_div(key, a.by_page);
        pg = t.table[col];
        in = key - col * a.page;
        if ((unsigned)pg >= (unsigned)a.pages) pg = -1;
      }
      float s = -INFINITY;
      if (pg >= 0) {
        const T* k = (const T*)a.k + pg * a.k_ps + in * a.k_rs + t.g * a.k_hs;
        s = 0.f;
        for (int d = 0; d < a.width; ++d) s += q_s[d] * Cvt<T>::ld(k + d);
        s *= c;
      }
      const float to = fmaxf(m, wave_max(s)), base = to == -INFINITY ? 0.f : to;
      const float p = pg >= 0 ? __builtin_amdgcn_exp2f(s - base) : 0.f, alpha = __builtin_amdgcn_exp2f(m - base);
      l = l * alpha + wave_sum(p);
      m = to;
#pragma unroll
      for (int j = 0; j < W / 64; ++j) acc[j] *= alpha;
      for (int u = 0; u < 64; ++u) {
        const int up = __shfl(pg, u, 64), ui = __shfl(in, u, 64);
        const float pu = __shfl(p, u, 64);
        if (up < 0) continue;
        const T* v = (const T*)a.v + up * a.v_ps + ui * a.v_rs + t.g * a.v_hs;
#pragma unroll
        for (int j = 0; j < W / 64; ++j)
          if (lane + 64 * j < a.width) acc[j] += pu * Cvt<T>::ld(v + lane + 64 * j);
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    if (slot >= 0) {
      const long long at = (long long)slot * f.slot_rows + rr;
#pragma unroll
      for (int j = 0; j < W / 64; ++j) f.part[at * W + lane + 64 * j] = acc[j];
      if (lane == 0) {
        f.ml[at * 2] = m;
        f.ml[at * 2 + 1] = l;
      }
    } else {
      T* o = (T*)a.o + row_offset(f, t, row, a.o_ts, a.o_hs);
#pragma unroll
      for (int j = 0; j < W / 64; ++j)
        if (lane + 64 * j < a.width) Cvt<T>::st(o + lane + 64 * j, l != 0.f ? acc[j] * inv : 0.f);
    }
  }
}

// One wave's subtiles of few rows: every fourth from ks0 on. Returns whether they are a case for exact_rows().
template <typename T, int W, int RUN>
__device__ __forceinline__ bool few_loop(const PagedAttnArgs& a, const FastArgs& f, const Tile& t, int ks0, int k1, bool valid,
                                         char* kt, unsigned k_lds, int lane, u32x4 (&qf)[W / 16], RowState<W>& st) {
  constexpr int SUB = 32 * W * 2, NP = SUB / 1024;
  const int hh = lane >> 5;
  char* const vt = kt + SUB;
  const unsigned v_lds = k_lds + SUB;
  PageRows<W, NP, RUN> pr;
  pr.init(a, t.table, t.g, t.klo, t.khi, lane);
  bool partial = false;       // the subtile whose transfer was begun last
  if (ks0 < k1) {
    pr.fetch(ks0);
    pr.known(ks0);
    partial = !pr.whole(ks0);
    pr.template issue<false>(ks0, k_lds, f.stream);
    pr.template issue<true>(ks0, v_lds, f.stream);
  }
  load_row<W>(a, f, t, t.rows0 + (lane & 31), valid, hh, qf, st);
  bool rare = false;
  for (; ks0 < k1; ks0 += kFewStep) {
    const int next = ks0 + kFewStep;
    const bool more = next < k1;
    rare |= pr.gone;
    const bool mask = ks0 + 31 > t.p_first || ks0 + 32 > t.cap || (a.window > 0 && ks0 < t.p_last - a.window + 1);
    if (more) pr.fetch(next);
    // the keys of this subtile are in LDS, its values may be on their way (as one instruction per piece, if it is whole)
    const bool whole = RUN == 0 || !partial;
    if (whole) wait_dma_but<NP>();
    else wait_dma_but<0>();
    rare |= subtile<T, W>(
        kt, vt, ks0, mask, f.c, qf, st, lane,
        [&]() {
          wait_lds();         // the key fragments are in registers: their place takes the next subtile's
          if (more) {
            pr.known(next);
            partial = !pr.whole(next);
            pr.template issue<false>(next, k_lds, f.stream);
          }
        },
        [&]() {
          if (more && (RUN == 0 || !partial)) wait_dma_but<NP>();
          else wait_dma_but<0>();
        },
        [&]() {
          wait_lds();
          if (more) pr.template issue<true>(next, v_lds, f.stream);
        });
  }
  return rare;
}

// Few rows (at most 32) over keys [k0, k1), k0 a multiple of 32: subtile t belongs to wave t % 4, each wave has its own
// part of LDS and its own running state; merged at the end, to the output (slot < 0) or to a slot of the workspace.
// Leaves without a barrier behind its last reads of LDS.
template <typename T, int W, int RUN>
__device__ __forceinline__ void few_rows(const PagedAttnArgs& a, const FastArgs& f, const Tile& t, int k0, int k1, int slot,
                                         char* smem, unsigned lds0, float (&ml_s)[4][32][2]) {
  constexpr int ND = W / 32, SUB = 32 * W * 2, REGION = 2 * SUB;
  static_assert(REGION == 32 * W * 4, "a wave's two subtiles and its fp32 output share their place");
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));      // opaque: what follows from it is computed per run, not kept across the runs
  const int lane = tid & 63, r32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const kt = smem + wave * REGION;
  const unsigned k_lds = lds0 + wave * REGION;
  u32x4 qf[W / 16];
  RowState<W> st;
  const bool valid = r32 < t.nrows;
  const bool rare = few_loop<T, W, RUN>(a, f, t, k0 + wave * 32, k1, valid, kt, k_lds, lane, qf, st);
  // ---- merge the waves ----
  const float l = sum_halves(st.l);
  if (hh == 0) {
    ml_s[wave][r32][0] = st.mb;
    ml_s[wave][r32][1] = l;
  }
  if (__syncthreads_or(rare)) {
    exact_rows<T, W>(a, f, t, k0, k1, slot, reinterpret_cast<float*>(smem));
    return;
  }
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (ml_s[w][r32][1] != 0.f) M = fmaxf(M, ml_s[w][r32][0]);
  const float scale = l != 0.f ? __builtin_amdgcn_exp2f(st.mb - M) : 0.f;
  if (valid) {
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = l != 0.f ? st.o[dt][4 * g4 + e] * scale : 0.f;
        *reinterpret_cast<f32x4*>(o_piece<W>(kt, r32, 8 * dt + 2 * g4 + hh)) = v;
      }
  }
  __syncthreads();
  for (int i = tid; i < t.nrows * (W / 8); i += kThreads) {
    const int rr = i / (W / 8), d8 = i % (W / 8);
    float M2 = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (ml_s[w][rr][1] != 0.f) M2 = fmaxf(M2, ml_s[w][rr][0]);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (ml_s[w][rr][1] != 0.f) L += ml_s[w][rr][1] * __builtin_amdgcn_exp2f(ml_s[w][rr][0] - M2);
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(o_piece<W>(smem + w * REGION, rr, 2 * d8));
      const f32x4 y = *reinterpret_cast<const f32x4*>(o_piece<W>(smem + w * REGION, rr, 2 * d8 + 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] += x[e];
        o[4 + e] += y[e];
      }
    }
    if (slot >= 0) {
      const long long at = (long long)slot * f.slot_rows + rr;
      store8(f.part + at * W + 8 * d8, o);
      if (d8 == 0) {
        f.ml[at * 2] = M2;
        f.ml[at * 2 + 1] = L;
      }
    } else if (8 * d8 < a.width) {
      const float inv = L != 0.f ? 1.f / L : 0.f;
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = L != 0.f ? Frag<T>::pack(o[2 * e] * inv, o[2 * e + 1] * inv) : 0u;
      *reinterpret_cast<u32x4*>((uint16_t*)a.o + row_offset(f, t, t.rows0 + rr, a.o_ts, a.o_hs) + 8 * d8) = w;
    }
  }
}

// `all`: cu_q says nothing about which rows belong to a request.
__device__ __forceinline__ void zero_rows_outside(const PagedAttnArgs& a, bool all = false) {
  const bool none = all || a.R == 0;
  const int lo = none ? a.N : min(max(a.cu_q[0], 0), a.N), hi = none ? a.N : min(max(a.cu_q[a.R], 0), a.N);
  const int rest = lo + a.N - max(hi, lo);
  const long long total = (long long)rest * a.nh * a.width;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
    const int d = (int)(i % a.width), h = (int)((i / a.width) % a.nh);
    int row = (int)(i / a.width / a.nh);
    if (row >= lo) row += max(hi, lo) - lo;
    ((uint16_t*)a.o)[(long long)row * a.o_ts + (long long)h * a.o_hs + d] = 0;
  }
}

// What the second kernel needs to know of a slot: the pieces of its tile if it holds the first of them (0: it does not),
// the tile, and where the others are: slot, then next + p * stride for p = 1 .. np - 1.
__device__ __forceinline__ void write_meta(const FastArgs& f, int slot, int np, int start, int rows0, int nrows, int g, int next,
                                           int stride) {
  int* m = f.meta + (long long)slot * 8;
  m[0] = np;
  m[1] = start;
  m[2] = rows0;
  m[3] = nrows;
  m[4] = g;
  m[5] = next;
  m[6] = stride;
}

template <typename T, int W, int RUN>
__global__ __launch_bounds__(kThreads, W == 64 ? 3 : 2) void paged_attn_few_kernel(PagedAttnArgs a, FastArgs f) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float ml_s[4][32][2];
  const int tid = threadIdx.x;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void*)smem;
  if (a.zero_rest) zero_rows_outside(a);
  __shared__ Runs runs;
  const int total = list_runs(a, f, runs);
  const int id = blockIdx.x;
  const int eff = min((int)gridDim.x, max(total, 1));
  const int per = max((total + eff - 1) / eff, 1);
  if (id == 0 && tid == 0) f.header[0] = 2 * eff;
  if (id >= eff) return;
  if (tid == 0) f.meta[(long long)(2 * id) * 8] = f.meta[(long long)(2 * id + 1) * 8] = 0;
  int at = id * per;
  const int end = min(at + per, total);
  for (bool first_run = true; at < end; first_run = false) {
    int first;
    Request q;
    const int r = find_run(a, f, runs, at, first, q);
    if (r < 0) break;
    const int steps = run_steps(q);
    if (steps == 0) break;
    const int run = (at - first) / steps, s0 = at - first - run * steps, s1 = min(steps, s0 + end - at);
    const int g = run % a.nkv, rows0 = run / a.nkv * kFewRows;
    if (s0 < 0 || run < 0 || rows0 >= q.rows) break;   // (count_items' bounds: never)
    const Tile t = make_tile(a, f, q, r, g, rows0, kFewRows);
    const int base = run_base(q), k0 = base + s0 * kFewStep, k1 = min(t.khi, base + s1 * kFewStep);
    const bool whole = s0 == 0 && s1 == steps;
    const int slot = whole ? -1 : 2 * id + (first_run ? 0 : 1);
    if (!first_run) __syncthreads();                  // the last run's outputs have been read from LDS
    few_rows<T, W, RUN>(a, f, t, k0, k1, slot, smem, lds0, ml_s);
    if (!whole && s0 == 0 && tid == 0) {
      const int last = min((at + steps - 1) / per, eff - 1);        // the workgroup that has its end
      write_meta(f, slot, last - id + 1, t.start, rows0, t.nrows, g, 2 * id, 2);
    }
    at += s1 - s0;
  }
}

// 128 rows over keys [k0, k1), k0 a multiple of 64: the waves share 64-key tiles. Returns whether they are a case for
// exact_rows().
template <typename T, int W, int RUN>
__device__ __forceinline__ bool chunk_loop(const PagedAttnArgs& a, const FastArgs& f, const Tile& t, int k0, int k1,
                                           char* smem, unsigned lds0, int wave, int lane, u32x4 (&qf)[W / 16], RowState<W>& st) {
  constexpr int SUB = 32 * W * 2, NP = 2 * SUB / 1024 / 4, STAGE = 4 * SUB;   // transfers per wave and tile; a K and a V tile
  const int r32 = lane & 31, hh = lane >> 5;
  PageRows<W, NP, RUN> pr;
  pr.init(a, t.table, t.g, t.klo, t.khi, lane);
  const int w_off = wave * 16;                               // the 16 rows of a tile that the wave transfers
  const unsigned w_lds = lds0 + wave * NP * 1024;
  bool rare = false;
  auto request_tile = [&](int at, int stage) {
    pr.known(at + w_off);
    rare |= pr.gone;
    pr.template issue<false>(at + w_off, w_lds + stage * STAGE);
    pr.template issue<true>(at + w_off, w_lds + stage * STAGE + 2 * SUB);
  };
  if (k0 < k1) {
    pr.fetch(k0 + w_off);
    request_tile(k0, 0);
  }
  const int row = t.rows0 + wave * 32;
  load_row<W>(a, f, t, row + r32, row + r32 < t.rows, hh, qf, st);
  const int wp_first = t.start + fast_div(min(row, t.rows - 1), f.by_group) + t.shift;
  const int wp_last = t.start + fast_div(min(row + 31, t.rows - 1), f.by_group) + t.shift;
  const bool wave_live = row < t.rows;
  int stage = 0;
  for (int kt0 = k0; kt0 < k1; kt0 += 64) {
    const int next = kt0 + 64;
    if (next < k1) pr.fetch(next + w_off);      // (under the wait for this tile)
    wait_dma_but<0>();
    __syncthreads();        // the tile has landed for every wave; every wave is done with the other stage
    if (next < k1) request_tile(next, stage ^ 1);      // (two ahead, in a third stage: no difference)
    const char* const kt = smem + stage * STAGE;
    const char* const vt = kt + 2 * SUB;
    stage ^= 1;
    if (!wave_live) continue;
#pragma unroll 1
    for (int ks0 = kt0; ks0 < kt0 + 64; ks0 += 32) {
      if (ks0 > wp_last || ks0 >= t.khi) break;
      if (a.window > 0 && ks0 + 31 < wp_first - a.window + 1) continue;
      const bool mask = ks0 + 31 > wp_first || ks0 + 32 > t.cap || (a.window > 0 && ks0 < wp_last - a.window + 1);
      const int at = (ks0 - kt0) * W * 2;
      rare |= chunk_tile<T, W>(kt + at, vt + at, ks0, mask, f.c, qf, st, lane);
    }
  }
  return rare;
}

// Chunks, with few-row requests among them. Four workgroups on a CU at width 64 (8 x 2048 rows of 16 heads 124 -> 121 us;
// two: 157), unless lanes hold addresses of their own (RUN 0), which takes the registers.
template <typename T, int W, int RUN>
__global__ __launch_bounds__(kThreads, W == 64 ? (RUN > 0 ? 4 : 3) : 2) void paged_attn_kernel(PagedAttnArgs a, FastArgs f) {
  constexpr int ND = W / 32, SUB = 32 * W * 2, REGION = 2 * SUB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float ml_s[4][32][2];
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void*)smem;
  if (a.zero_rest) zero_rows_outside(a);

  // ---- this workgroup's item ----
  const Item it = find_item(a, f, blockIdx.x, lane);
  const int r = __builtin_amdgcn_readfirstlane(it.r);
  if (r < 0) return;
  const Request q = request(a, f.G, r);
  const int np = __builtin_amdgcn_readfirstlane(it.np);
  int slot = __builtin_amdgcn_readfirstlane(it.slot);
  int j = __builtin_amdgcn_readfirstlane(it.j);
  const int g = j % a.nkv;
  j /= a.nkv;
  const int piece = j % np;
  const int tile = q.tiles - 1 - j / np;                 // the rows that see most come first
  if (tile < 0 || j < 0 || (np > 1 && (unsigned)slot >= (unsigned)f.max_slots)) return;   // (count_items' bounds: never)
  const int rows0 = tile * kChunkRows;
  const Tile t = make_tile(a, f, q, r, g, rows0, q.chunk ? kChunkRows : kFewRows);
  const int nrows = t.nrows, step = q.chunk ? kChunkStep : kFewStep;
  const int k_base = t.klo & ~63;
  const int span = ((t.khi - k_base + np - 1) / np + step - 1) / step * step;
  const int k0 = k_base + piece * span, k1 = min(t.khi, k0 + span);
  if (np > 1 && tid == 0) write_meta(f, slot, piece == 0 ? np : 0, q.start, rows0, nrows, g, slot, a.nkv);
  if (!q.chunk) {
    few_rows<T, W, RUN>(a, f, t, k0, k1, np > 1 ? slot : -1, smem, lds0, ml_s);
    return;
  }

  u32x4 qf[W / 16];
  RowState<W> st;
  // (a barrier too: every wave is done with the tiles)
  if (__syncthreads_or(chunk_loop<T, W, RUN>(a, f, t, k0, k1, smem, lds0, wave, lane, qf, st))) {
    exact_rows<T, W>(a, f, t, k0, k1, np > 1 ? slot : -1, reinterpret_cast<float*>(smem));
    return;
  }
  const float l = sum_halves(st.l);
  char* const tile_o = smem + wave * REGION;
  const float inv = np > 1 ? 1.f : (l != 0.f ? 1.f / l : 0.f);
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = l != 0.f ? st.o[dt][4 * g4 + e] * inv : 0.f;
      *reinterpret_cast<f32x4*>(o_piece<W>(tile_o, r32, 8 * dt + 2 * g4 + hh)) = v;
    }
  wait_lds();
  const int mine = min(32, nrows - wave * 32);
  for (int i = lane; i < mine * (W / 8); i += 64) {
    const int rr = i / (W / 8), d8 = i % (W / 8), rw = wave * 32 + rr;
    const f32x4 x = *reinterpret_cast<const f32x4*>(o_piece<W>(tile_o, rr, 2 * d8));
    const f32x4 y = *reinterpret_cast<const f32x4*>(o_piece<W>(tile_o, rr, 2 * d8 + 1));
    if (np > 1) {
      float* dst = f.part + ((long long)slot * f.slot_rows + rw) * W + 8 * d8;
      *reinterpret_cast<f32x4*>(dst) = x;
      *reinterpret_cast<f32x4*>(dst + 4) = y;
    } else if (8 * d8 < a.width) {
      const u32x4 w = {Frag<T>::pack(x[0], x[1]), Frag<T>::pack(x[2], x[3]), Frag<T>::pack(y[0], y[1]), Frag<T>::pack(y[2], y[3])};
      *reinterpret_cast<u32x4*>((uint16_t*)a.o + row_offset(f, t, rows0 + rw, a.o_ts, a.o_hs) + 8 * d8) = w;
    }
  }
  if (np > 1 && hh == 0 && r32 < mine) {
    const long long at = (long long)slot * f.slot_rows + wave * 32 + r32;
    f.ml[at * 2] = st.mb;
    f.ml[at * 2 + 1] = l;
  }
}

// The pieces of one row tile and KV head: o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p. A workgroup takes kJoinRows
// rows; a thread has 8 columns of a row and every `groups`-th piece, four of them requested together, and the groups are
// joined through LDS: always in the same order.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void paged_attn_join_kernel(PagedAttnArgs a, FastArgs f) {
  constexpr int CPR = W / 8, kJoinRows = kThreads / CPR, U = 4;
  __shared__ float o_s[kThreads][9], m_s[kThreads];      // (9: rows of 8 floats would share banks)
  const int slot = blockIdx.x;
  if (f.header[3] != 0) {       // nothing was computed
    if (a.zero_rest) zero_rows_outside(a, true);
    return;
  }
  if (slot >= f.header[0]) return;
  const int* meta = f.meta + (long long)slot * 8;
  const int np = meta[0], start = meta[1], rows0 = meta[2], nrows = min(meta[3] - (int)blockIdx.y * kJoinRows, kJoinRows), g = meta[4];
  const int other = meta[5], stride = meta[6];
  if (np < 2 || nrows <= 0 || other + (np - 1) * stride >= f.max_slots) return;
  const int row_b = blockIdx.y * kJoinRows, units = nrows * CPR;
  int groups = 1;
  while (2 * groups * units <= kThreads) groups *= 2;
  const int tid = threadIdx.x, unit = tid % units, grp = tid / units;
  const int rr = row_b + unit / CPR, d8 = unit % CPR;
  float M = -INFINITY, L = 0.f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  if (grp < groups) {
    for (int p0 = grp; p0 < np; p0 += groups * U) {
      float m[U], l[U], x[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int p = min(p0 + u * groups, np - 1);
        const long long at = (long long)(p == 0 ? slot : other + p * stride) * f.slot_rows + rr;
        m[u] = f.ml[at * 2];
        l[u] = p0 + u * groups < np ? f.ml[at * 2 + 1] : 0.f;
        load8(f.part + at * W + 8 * d8, x[u]);
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (l[u] != 0.f) top = fmaxf(top, m[u]);
      const float keep = L != 0.f ? __builtin_amdgcn_exp2f(M - top) : 0.f;
      L *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (l[u] != 0.f) {
          const float w = __builtin_amdgcn_exp2f(m[u] - top);
          L += l[u] * w;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] += x[u][e] * w;
        }
      M = top;
    }
    m_s[tid] = M;
#pragma unroll
    for (int e = 0; e < 8; ++e) o_s[tid][e] = o[e];
    o_s[tid][8] = L;
  }
  __syncthreads();
  if (grp != 0 || 8 * d8 >= a.width) return;
  for (int w = 1; w < groups; ++w) {
    const int t = unit + w * units;
    const float m = m_s[t], l = o_s[t][8];
    if (l == 0.f) continue;
    const float top = fmaxf(M, m), keep = L != 0.f ? __builtin_amdgcn_exp2f(M - top) : 0.f, add = __builtin_amdgcn_exp2f(m - top);
    L = L * keep + l * add;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * keep + o_s[t][e] * add;
    M = top;
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = L != 0.f ? Frag<T>::pack(o[2 * e] * inv, o[2 * e + 1] * inv) : 0u;
  const int tk = fast_div(rows0 + rr, f.by_group), hd = g * f.G + rows0 + rr - tk * f.G;
  *reinterpret_cast<u32x4*>((uint16_t*)a.o + (long long)(start + tk) * a.o_ts + (long long)hd * a.o_hs + 8 * d8) = w;
}

// Whether the matrix kernels take the call: 16-bit types, whole aligned 16-byte pieces, offsets inside a page below 2^31.
bool fast_ok(const PagedAttnArgs& a) {
  if (a.type == kTypeFloat || a.width % 8 != 0 || a.width > 128) return false;
  const long long strides[] = {a.q_ts, a.q_hs, a.o_ts, a.o_hs, a.k_ps, a.k_rs, a.k_hs, a.v_ps, a.v_rs, a.v_hs};
  for (long long s : strides)
    if (s % 8 != 0 || s < 0) return false;
  for (const void* p : {a.q, a.k, a.v, (const void*)a.o})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  const long long lim = 1ll << 31;
  return a.k_rs * 2 * std::max(a.page, 16) < lim && a.v_rs * 2 * std::max(a.page, 16) < lim && a.k_ps * 2 < lim && a.v_ps * 2 < lim;
}

struct Plan : Counts {
  size_t part, ml, meta, total;
};
Plan plan_items(const PagedAttnArgs& a, int num_cus) {
  Plan p{count_items(a, num_cus)};
  const int W = a.width <= 64 ? 64 : 128;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  p.part = up((size_t)p.slots * p.slot_rows * W * 4);
  p.ml = up((size_t)p.slots * p.slot_rows * 8);
  p.meta = up((size_t)p.slots * 32);
  p.total = p.part + p.ml + p.meta + 256 + (a.R > kWaveRequests ? up((size_t)(a.R + 1) * 12) : 0);
  return p;
}

template <typename T, int W, int RUN, bool CHUNKS>
void launch_fast(const PagedAttnArgs& a, const FastArgs& f, int grid, hipStream_t st) {
  constexpr int lds = 4 * 2 * 32 * W * 2;
  auto kernel = CHUNKS ? paged_attn_kernel<T, W, RUN> : paged_attn_few_kernel<T, W, RUN>;
  static bool set[64] = {};      // by device: above the default limit of dynamic LDS, the same value every time
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64 || !set[dev]) {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  if (a.R > kWaveRequests) hipLaunchKernelGGL((paged_attn_items_kernel<CHUNKS>), dim3(1), dim3(1024), 0, st, a, f);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), lds, st, a, f);
  hipLaunchKernelGGL((paged_attn_join_kernel<T, W>), dim3(f.max_slots, (f.slot_rows * (W / 8) + kThreads - 1) / kThreads),
                     dim3(kThreads), 0, st, a, f);
}
template <typename T, int W>
void launch_fast(const PagedAttnArgs& a, const FastArgs& f, const Plan& p, hipStream_t st) {
  const int run = a.width != W ? 0 : a.page % 16 == 0 ? 16 : a.page % (512 / W) == 0 ? 512 / W : 0;
  if (p.chunks) {
    if (run == 16) launch_fast<T, W, 16, true>(a, f, p.grid, st);
    else if (run > 0) launch_fast<T, W, 512 / W, true>(a, f, p.grid, st);
    else launch_fast<T, W, 0, true>(a, f, p.grid, st);
  } else {
    if (run == 16) launch_fast<T, W, 16, false>(a, f, p.grid, st);
    else if (run > 0) launch_fast<T, W, 512 / W, false>(a, f, p.grid, st);
    else launch_fast<T, W, 0, false>(a, f, p.grid, st);
  }
}

}  // namespace

size_t paged_attn_workspace(const PagedAttnArgs& a, int num_cus) {
  return a.N > 0 && a.R > 0 && fast_ok(a) ? plan_items(a, num_cus).total : 0;
}

void paged_attn(const PagedAttnArgs& a, int num_cus, void* workspace, hipStream_t st) {
  if (a.N == 0 || a.nh == 0) return;
  if (workspace != nullptr) {
    const Plan p = plan_items(a, num_cus);
    FastArgs f{};
    f.negate = a.scale < 0.f;
    f.c = std::max(std::fabs(a.scale) * kLog2e, 1e-30f);      // a scale of 0: equal weights, and no 0 * inf at masked keys
    f.G = a.nh / a.nkv;
    f.by_group = make_fast_div(f.G);
    f.target = p.target;
    // measured: 64 x 8k 265 -> 248 us, 2 x 128k 131 -> 124 us; a small cache may still be there for the next step
    f.stream = 4ll * a.pages * a.page * a.nkv * a.width >= stream_threshold_bytes();
    f.max_slots = p.slots;
    f.slot_rows = p.slot_rows;
    char* w = (char*)workspace;
    f.part = (float*)w;
    f.ml = (float*)(w + p.part);
    f.meta = (int*)(w + p.part + p.ml);
    f.header = (int*)(w + p.part + p.ml + p.meta);
    f.prefix = f.header + 64;
    const bool bf = a.type == kTypeBf16;
    if (a.width <= 64) bf ? launch_fast<bf16_t, 64>(a, f, p, st) : launch_fast<half_t, 64>(a, f, p, st);
    else bf ? launch_fast<bf16_t, 128>(a, f, p, st) : launch_fast<half_t, 128>(a, f, p, st);
    return;
  }
  const long long waves = (long long)a.N * a.nh;
  const long long groups = (waves + kGenWaves - 1) / kGenWaves, gx = std::min(groups, 1ll << 20);
  const dim3 grid((unsigned)gx, (unsigned)((groups + gx - 1) / gx)), block(kGenWaves * 64);
  if (a.type == kTypeBf16) hipLaunchKernelGGL((paged_attn_rows_kernel<bf16_t>), grid, block, 0, st, a);
  else if (a.type == kTypeHalf) hipLaunchKernelGGL((paged_attn_rows_kernel<half_t>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged_attn_rows_kernel<float>), grid, block, 0, st, a);
}

}  // namespace dpa
