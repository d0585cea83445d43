// How paged attention cuts a ragged batch into work (csrc/paged_attn.hip): arithmetic on the requests' lengths that the
// kernels, their launcher and the host-side checks share. Plain C++ apart from DPA_HD, so it builds with g++ as well.
// Args is PagedAttnArgs or a stand-in with its cu_q, kv_lens, N, R, M, page, window, nh, nkv, width and max_q.
#pragma once
#include "host_logic.h"

namespace dpa {
namespace paged {

constexpr int kFewRows = 32, kChunkRows = 128;
constexpr int kFewStep = 128, kChunkStep = 64;      // keys a workgroup advances by: pieces are multiples of it
constexpr int kWaveRequests = 256;    // up to here every wave derives the items by itself

DPA_HD int imin(int a, int b) { return a < b ? a : b; }
DPA_HD int imax(int a, int b) { return a > b ? a : b; }

struct Request {
  int start, n;        // its rows of the batch
  int shift;           // position of batch row i: i + shift
  int rows, tiles;     // packed rows per KV head and tiles of them
  int klo, khi;        // keys that any of its rows sees
  bool chunk;
  bool back;           // cu_q decreases here
};
template <class Args>
DPA_HD void key_range(const Args& a, Request& q) {
  q.klo = a.window > 0 ? imax(q.start + q.shift - a.window + 1, 0) : 0;
  q.khi = imax(imin(q.start + q.n + q.shift, a.M * a.page), q.klo);
}
template <class Args>
DPA_HD Request request(const Args& a, int G, int r) {
  Request q;
  const int c0 = a.cu_q[r], c1 = a.cu_q[r + 1];
  q.start = imin(imax(c0, 0), a.N);
  q.n = imin(imax(c1, q.start), a.N) - q.start;
  q.back = c1 < c0;
  const long long sh = (long long)a.kv_lens[r] - c1, most = 1ll << 30;
  q.shift = (int)(sh < -most ? -most : sh > most ? most : sh);
  q.rows = q.n * G;
  q.chunk = q.rows > kFewRows;
  q.tiles = q.chunk ? (q.rows + kChunkRows - 1) / kChunkRows : (q.rows > 0 ? 1 : 0);
  key_range(a, q);
  return q;
}

// Work of a request: keys walked by a workgroup, those of a chunk counted twice (its steps have 64 keys, those of few
// rows 128).
DPA_HD float request_cost(const Request& q) { return (float)q.tiles * (float)(q.khi - q.klo) * (q.chunk ? 2.f : 1.f); }
struct PieceSize {
  int few, chunk;      // keys
};
// (the limits are 2.05e9 keys, past the 2^30 of the longest request: what they cut is one piece)
DPA_HD PieceSize piece_size(float cost, int nkv, int target) {
  const float budget = cost * (float)nkv / (float)target;
  const float few = budget / (float)kFewStep, chunk = budget * 0.5f / (float)kChunkStep;
  PieceSize p;
  p.few = imax((int)(few < 1.6e7f ? few : 1.6e7f) + 1, 2) * kFewStep;
  p.chunk = imax((int)(chunk < 3.2e7f ? chunk : 3.2e7f) + 1, 8) * kChunkStep;
  return p;
}
DPA_HD int pieces(const Request& q, const PieceSize& p) {
  const int len = q.khi - q.klo, step = q.chunk ? p.chunk : p.few;
  return len <= step ? 1 : (len + step - 1) / step;
}
// Items of a request in the list's two passes, the later tiles first.
DPA_HD int first_items(const Request& q, int np, int nkv) { return (q.tiles - q.tiles / 3) * np * nkv; }
DPA_HD int second_items(const Request& q, int np, int nkv) { return q.tiles / 3 * np * nkv; }

// Few rows: 128-key steps of a run, and runs of a request.
DPA_HD int run_base(const Request& q) { return q.klo & ~31; }
DPA_HD int run_steps(const Request& q) {
  return q.rows > 0 ? imax((q.khi - run_base(q) + kFewStep - 1) / kFewStep, 1) : 0;
}
DPA_HD int run_count(const Request& q, int nkv) { return (q.rows + kFewRows - 1) / kFewRows * nkv; }

// What the host fixes without knowing the lengths. It holds for every cu_q that does not decrease: the requests' rows are
// then disjoint, so that there are at most `target` + tiles * nkv items, as many slots as two per `target` and, of few
// rows, fewer than 2^30 steps. The kernels compute nothing for a cu_q that decreases anywhere.
struct Counts {
  int target, grid, slots, slot_rows;
  bool chunks;
};
template <class Args>
inline Counts count_items(const Args& a, int num_cus) {
  Counts p;
  const int G = a.nh / a.nkv;
  const long long most = 1ll << 30;
  // (the 128-key steps of all runs are counted in 32 bits; pages shared by many long requests could pass that)
  const long long steps = (a.R + (long long)a.N * G / kFewRows) * a.nkv * ((long long)a.M * a.page / kFewStep + 2);
  p.chunks = ((long long)a.N * G > kFewRows && (long long)a.max_q * G > kFewRows) || steps >= most;
  if (p.chunks) {
    p.target = num_cus * 2;         // (4: 43 instead of 37 us on a mixed batch of 33 requests, no difference on prompts)
    // tiles: one per request with rows, and one more for every 128 rows of a chunk
    const long long tiles = (a.N < a.R ? a.N : a.R) + (long long)a.N * G / kChunkRows;
    const long long grid = p.target + tiles * a.nkv;
    p.grid = (int)(grid < most ? grid : most);
    p.slots = imin(2 * p.target, p.grid);
    p.slot_rows = kChunkRows;
  } else {
    p.target = 0;
    p.grid = num_cus * (a.width <= 64 ? 3 : 2);      // the workgroups that fit the card at once
    p.slots = 2 * p.grid;
    p.slot_rows = kFewRows;
  }
  return p;
}

}  // namespace paged
}  // namespace dpa
