// Page tables and slot maps of a ragged batch, built on the device from the requests' lengths (gfx950).
//
//   cu[r + 1]   = min(cu[r] + max(q[r], 0), N)            cu[0] = 0; requests past N rows are cut there
//   kv[r]       = c[r] + n[r],  n[r] = cu[r + 1] - cu[r]   rows in the cache after the step
//   have[r]     = min(ceil(c[r] / p), M)                   table columns already filled
//   need[r]     = max(min(ceil(kv[r] / p), M) - have[r], 0), first[r] = sum of need below r
//   table[r, have[r] + j] = F[f - 1 - (first[r] + j)]      pages come off the end of the free list; -1 when it is empty
//   row i of request r: position c[r] + i - cu[r], slot = table[r, position / p] * p + position % p (-1: no page)
//
// One launch, no pass over memory between its parts: a workgroup owns 1024 rows of the batch and runs the two prefix
// sums over ALL requests itself (R is a few thousand at most: 16 KB from L2 at R = 2048), which costs less than a
// second launch. While it walks the requests, the thread that owns one whose rows reach into the block's range leaves
// the request's numbers in LDS at the first such row; a running maximum over the rows then tells every row its
// request. A row never reads a table entry that this launch writes: pages at or past have[r] come straight from the
// free list. Both sums saturate at N, so int32 holds them whatever the lengths say. Bound by latency: 64 requests and
// rows 5.6 us (7.5 us a call from Python), 4096 requests and 512 K rows 12.0 us (13.5 without the next scan's lengths
// requested ahead; 1024 threads and one scan: 16.5).
#include "paged.h"

namespace dpa {

namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanPer = 4;                             // requests per thread and scan, rows per thread
constexpr int kPlanRows = kPlanThreads * kPlanPer;      // rows of the batch per workgroup
constexpr int kMaxLen = 1 << 30;

// Exclusive prefix of v over the workgroup under sat(a + b) = min(a + b, cap), cap < 2^30; total: over all threads.
__device__ __forceinline__ int scan_sat(int v, int cap, int* red, int& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(incl, off, 64);
    if (lane >= off) incl = min(incl + o, cap);
  }
  __syncthreads();
  if (lane == 63) red[wid] = incl;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wid) base = min(base + red[w], cap);
    all = min(all + red[w], cap);
  }
  total = all;
  const int left = __shfl_up(incl, 1, 64);
  return lane == 0 ? base : min(base + left, cap);
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedPlanArgs a) {
  __shared__ int red[kPlanThreads / 64];
  __shared__ int s_req[kPlanRows], s_cu[kPlanRows], s_ctx[kPlanRows], s_first[kPlanRows];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int i0 = blockIdx.x * kPlanRows;
  const int p = a.page, N = a.tokens;
  for (int i = tid; i < kPlanRows; i += kPlanThreads) s_req[i] = -1;
  const int count = min(max(*a.free_count, 0), a.free_cap);

  int carry_q = 0, carry_p = 0, wanted = 0;
  int next_q[kPlanPer], next_c[kPlanPer];      // the next scan's lengths, requested before this one's barriers
  auto request = [&](int r0) {
#pragma unroll
    for (int j = 0; j < kPlanPer; ++j) {
      const int r = r0 + tid * kPlanPer + j;
      next_q[j] = r < a.R ? a.q_lens[r] : 0;
      next_c[j] = r < a.R ? a.ctx_lens[r] : 0;
    }
  };
  request(0);
  for (int r0 = 0, pass = 0; r0 < a.R; r0 += kPlanRows, ++pass) {
    const int rb = r0 + tid * kPlanPer;
    int q[kPlanPer], c[kPlanPer], sum = 0;
#pragma unroll
    for (int j = 0; j < kPlanPer; ++j) {
      q[j] = min(max(next_q[j], 0), N);
      c[j] = min(max(next_c[j], 0), kMaxLen);
      sum = min(sum + q[j], N);
    }
    if (r0 + kPlanRows < a.R) request(r0 + kPlanRows);
    int total;
    int cu = min(carry_q + scan_sat(sum, N, red, total), N);
    carry_q = min(carry_q + total, N);
    int need[kPlanPer], cus[kPlanPer], have[kPlanPer];
    sum = 0;
#pragma unroll
    for (int j = 0; j < kPlanPer; ++j) {
      cus[j] = cu;
      const int next = min(cu + q[j], N);
      q[j] = next - cu;
      cu = next;
      const int had = fast_div(c[j] + p - 1, a.by_page), want = fast_div(c[j] + q[j] + p - 1, a.by_page);
      wanted += want - had;
      have[j] = min(had, a.M);
      need[j] = min(want, a.M) - have[j];
      sum += need[j];      // a new page holds a new row, so the sum stays within N
    }
    int first = carry_p + scan_sat(sum, N, red, total);
    carry_p += total;
    const bool writer = pass % gridDim.x == blockIdx.x;
#pragma unroll
    for (int j = 0; j < kPlanPer; ++j) {
      if (writer && rb + j < a.R) {
        a.cu_q[rb + j + 1] = cus[j] + q[j];
        a.kv_lens[rb + j] = c[j] + q[j];
      }
      if (q[j] > 0 && cus[j] < i0 + kPlanRows && cus[j] + q[j] > i0) {
        const int s = max(cus[j], i0) - i0;
        s_req[s] = rb + j;
        s_cu[s] = cus[j];
        s_ctx[s] = c[j];
        s_first[s] = first - have[j];
      }
      first += need[j];
    }
  }
  if (blockIdx.x == 0) {
    int all;
    scan_sat(wanted, N, red, all);
    if (tid == 0) {
      a.cu_q[0] = 0;
      const int had = min(carry_p, count);
      a.free_left[0] = count - had;
      a.free_left[1] = all - had;
    }
  }
  __syncthreads();

  // the last marked row at or before each row
  const int t0 = tid * kPlanPer;
  int mark[kPlanPer], m = -1;
#pragma unroll
  for (int j = 0; j < kPlanPer; ++j) {
    if (s_req[t0 + j] >= 0) m = t0 + j;
    mark[j] = m;
  }
  int incl = m;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(incl, off, 64);
    if (lane >= off) incl = max(incl, o);
  }
  if (lane == 63) red[wid] = incl;
  __syncthreads();
  int before = __shfl_up(incl, 1, 64);
  if (lane == 0) before = -1;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w)
    if (w < wid) before = max(before, red[w]);
#pragma unroll
  for (int j = 0; j < kPlanPer; ++j) {
    const int i = i0 + t0 + j;
    if (i >= N) break;
    const int s = max(mark[j], before);
    int pos = 0, slot = -1;
    if (s >= 0 && i < carry_q) {
      const int r = s_req[s];
      pos = s_ctx[s] + i - s_cu[s];
      const int pg = fast_div(pos, a.by_page), off = pos - pg * p;
      if (pg < a.M) {
        int* entry = a.table + (long long)r * a.table_ld + pg;
        const int nth = s_first[s] + pg;   // how many-th page of this step; below have[r]: an old page
        int held;
        if (pg < min(fast_div(s_ctx[s] + p - 1, a.by_page), a.M)) held = *entry;
        else {
          held = nth < count ? a.free_pages[count - 1 - nth] : -1;
          if (off == 0) *entry = held;     // the first row of a new page is a new row
        }
        const long long at = (long long)held * p + off;
        if (held >= 0 && at < 0x7fffffffll) slot = (int)at;
      }
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
}

}  // namespace

void paged_plan(const PagedPlanArgs& a, hipStream_t st) {
  const int blocks = a.tokens > kPlanRows ? (a.tokens + kPlanRows - 1) / kPlanRows : 1;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, st, a);
}

}  // namespace dpa
