// New key / value rows into the pages of a KV cache (gfx950): row i goes to row slots[i] % page of page slots[i] / page.
//
// A copy with a scattered destination: bound by memory. Threads take 16-byte pieces (single elements where a stride, a
// width or an address does not allow them), kUnroll of them requested before the first is written. The new rows are
// read past the caches (nothing reads them again); the pages are written into them, since attention reads them next,
// unless the call alone is more than they hold. 32785 rows of 8 x 128 keys and values: 53 us (5.1 TB/s; 4 pieces at a
// time 60 us; a large copy runs at 4.9 TB/s).
#include "paged.h"

namespace dpa {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kUnroll = 2;

struct AppendMap {
  FastDiv by_token, by_khead, by_vhead;   // pieces per token (k and v), per key head, per value head
  int per_token, k_pieces, k_head, v_head;
};

template <typename P, bool NT>   // P: one piece; NT: written past the caches too
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(PagedAppendArgs a, AppendMap m, int tokens_per_block) {
  const int t0 = blockIdx.x * tokens_per_block;
  const int n = min(tokens_per_block, a.N - t0) * m.per_token;
  const int es = sizeof(P) / a.elem;   // elements per piece
  const int rows = a.pages * a.page;
  for (int base = threadIdx.x; base < n; base += kAppendThreads * kUnroll) {
    P val[kUnroll];
    P* dst[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int id = base + u * kAppendThreads;
      dst[u] = nullptr;
      if (id >= n) continue;
      const int t = fast_div(id, m.by_token), piece = id - t * m.per_token;
      const int slot = a.slots[t0 + t];
      if (slot < 0 || slot >= rows) continue;
      const int pg = fast_div(slot, a.by_page), row = slot - pg * a.page;
      const bool is_v = piece >= m.k_pieces;
      const int pc = is_v ? piece - m.k_pieces : piece;
      const int h = is_v ? fast_div(pc, m.by_vhead) : fast_div(pc, m.by_khead);
      const int e = (pc - h * (is_v ? m.v_head : m.k_head)) * es;
      const long long from = (long long)(t0 + t) * (is_v ? a.v_ts : a.k_ts) + h * (is_v ? a.v_hs : a.k_hs) + e;
      const long long to = is_v ? pg * a.vp_ps + row * a.vp_rs + h * a.vp_hs + e : pg * a.kp_ps + row * a.kp_rs + h * a.kp_hs + e;
      val[u] = __builtin_nontemporal_load(reinterpret_cast<const P*>((const char*)(is_v ? a.v : a.k) + from * a.elem));
      dst[u] = reinterpret_cast<P*>((char*)(is_v ? a.v_pages : a.k_pages) + to * a.elem);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (dst[u] != nullptr) {
        if (NT) __builtin_nontemporal_store(val[u], dst[u]);
        else *dst[u] = val[u];
      }
  }
}

template <typename P>
void launch_append(const PagedAppendArgs& a, hipStream_t st) {
  const int es = sizeof(P) / a.elem;
  AppendMap m;
  m.k_head = a.dk / es;
  m.v_head = a.dv / es;
  m.k_pieces = a.nkv * m.k_head;
  m.per_token = m.k_pieces + a.nkv * m.v_head;
  m.by_token = make_fast_div(m.per_token);
  m.by_khead = make_fast_div(m.k_head);
  m.by_vhead = make_fast_div(m.v_head);
  const int goal = kAppendThreads * kUnroll;
  const int tokens = m.per_token >= goal ? 1 : goal / m.per_token;
  const dim3 grid((a.N + tokens - 1) / tokens), block(kAppendThreads);
  if ((long long)a.N * m.per_token * (long long)sizeof(P) >= stream_threshold_bytes())
    hipLaunchKernelGGL((paged_append_kernel<P, true>), grid, block, 0, st, a, m, tokens);
  else
    hipLaunchKernelGGL((paged_append_kernel<P, false>), grid, block, 0, st, a, m, tokens);
}

}  // namespace

void paged_append(const PagedAppendArgs& a, hipStream_t st) {
  if (a.N == 0 || a.pages == 0) return;
  const int es = 16 / a.elem;
  auto ok = [&](const void* p, long long s0, long long s1, long long s2) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 % es == 0 && s1 % es == 0 && s2 % es == 0;
  };
  const bool wide = a.dk % es == 0 && a.dv % es == 0 && ok(a.k, a.k_ts, a.k_hs, 0) && ok(a.v, a.v_ts, a.v_hs, 0) &&
                    ok(a.k_pages, a.kp_ps, a.kp_rs, a.kp_hs) && ok(a.v_pages, a.vp_ps, a.vp_rs, a.vp_hs);
  if (wide) launch_append<u32x4>(a, st);
  else if (a.elem == 2) launch_append<uint16_t>(a, st);
  else launch_append<uint32_t>(a, st);
}

}  // namespace dpa
