// Host model of the work lists of paged attention over csrc/paged_items.h, built by tests/test_paged_items_cpu.py with
// g++ under AddressSanitizer + UBSan. For every batch of lengths: each item has a workgroup, each slot of the workspace
// that the joining kernel reads is written by exactly one item, and each row tile's keys are covered once.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <utility>
#include <vector>

#include "paged_items.h"

using namespace dpa::paged;

static int g_failed = 0;
#define CHECK(cond)                                                     \
  do {                                                                  \
    if (!(cond)) {                                                      \
      if (g_failed < 20) std::fprintf(stderr, "%s:%d: CHECK failed: %s\n", __FILE__, __LINE__, #cond); \
      ++g_failed;                                                       \
    }                                                                   \
  } while (0)

struct Batch {
  const int *cu_q, *kv_lens;
  int N, R, M, page, window, nh, nkv, width, max_q;
};
constexpr int kCus = 256;

// Chunks: ids in two passes over the requests, slots for what is cut. Returns the slots below header[0] that no launched
// item writes. guarded: offsets that decrease leave the list empty, as in the kernels.
static int chunk_list(const Batch& b, bool guarded) {
  const Counts c = count_items(b, kCus);
  const int G = b.nh / b.nkv;
  std::vector<Request> q(b.R);
  float cost = 0.f;
  bool back = false;
  for (int r = 0; r < b.R; ++r) {
    q[r] = request(b, G, r);
    cost += request_cost(q[r]);
    back |= q[r].back;
  }
  if (guarded && back) return 0;
  const PieceSize size = piece_size(cost, b.nkv, c.target);
  long long all1 = 0, slots = 0;
  std::vector<long long> first(b.R), slot0(b.R);
  for (int r = 0; r < b.R; ++r) {
    if (q[r].tiles == 0) continue;
    const int np = pieces(q[r], size);
    first[r] = all1;
    slot0[r] = slots;
    all1 += first_items(q[r], np, b.nkv);
    if (np > 1) slots += (long long)q[r].tiles * np * b.nkv;
  }
  const long long header = std::min<long long>(slots, c.slots);
  std::vector<char> written(header, 0);
  long long id2 = all1, lost = 0;
  for (int r = 0; r < b.R; ++r) {
    if (q[r].tiles == 0) continue;
    const int np = pieces(q[r], size), n1 = first_items(q[r], np, b.nkv), n2 = second_items(q[r], np, b.nkv);
    for (int j = 0; j < n1 + n2; ++j) {
      const long long id = j < n1 ? first[r] + j : id2 + j - n1;
      const long long slot = slot0[r] + j;
      if (id >= c.grid) { ++lost; continue; }
      const int tile = q[r].tiles - 1 - j / b.nkv / np;
      CHECK(tile >= 0);
      if (np > 1 && slot < header) {
        CHECK(!written[slot]);
        written[slot] = 1;
      } else if (np > 1) {
        ++lost;
      }
    }
    id2 += n2;
  }
  if (guarded) CHECK(lost == 0);
  return (int)std::count(written.begin(), written.end(), 0);
}

// Few rows: equal shares of all steps. Every (run, step) belongs to one workgroup, and what a first piece announces is there.
static void few_list(const Batch& b) {
  const Counts c = count_items(b, kCus);
  const int G = b.nh / b.nkv;
  std::vector<long long> before(b.R + 1, 0);
  std::vector<Request> q(b.R);
  for (int r = 0; r < b.R; ++r) {
    q[r] = request(b, G, r);
    if (q[r].back) return;
    before[r + 1] = before[r] + (long long)run_steps(q[r]) * run_count(q[r], b.nkv);
  }
  CHECK(before[b.R] < (1ll << 30));
  const int total = (int)before[b.R], eff = std::min(c.grid, std::max(total, 1)), per = std::max((total + eff - 1) / eff, 1);
  std::set<int> written;
  std::vector<std::pair<int, int>> joins;      // first slot, pieces
  long long steps_done = 0;
  for (int id = 0; id < eff; ++id) {
    int at = id * per;
    const int end = std::min(at + per, total);
    int cut = 0;
    for (bool first_run = true; at < end; first_run = false) {
      const int r = (int)(std::upper_bound(before.begin(), before.end(), (long long)at) - before.begin()) - 1;
      const int steps = run_steps(q[r]), first = (int)before[r];
      const int run = (at - first) / steps, s0 = at - first - run * steps, s1 = std::min(steps, s0 + end - at);
      CHECK(s0 >= 0 && run / b.nkv * kFewRows < q[r].rows);
      steps_done += s1 - s0;
      if (s0 != 0 || s1 != steps) {
        const int slot = 2 * id + (first_run ? 0 : 1);
        CHECK(written.insert(slot).second && ++cut <= 2 && slot < c.slots);
        if (s0 == 0) {
          const int last = std::min((at + steps - 1) / per, eff - 1);
          joins.push_back({slot, last - id + 1});
          CHECK(last > id);
        }
      }
      at += s1 - s0;
    }
  }
  CHECK(steps_done == total);
  size_t pieces_read = 0;
  for (const auto& j : joins)
    for (int p = 0; p < j.second; ++p, ++pieces_read) CHECK(written.count(p == 0 ? j.first : (j.first & ~1) + 2 * p));
  CHECK(pieces_read == written.size());
}

static Batch batch(const std::vector<int>& cu, const std::vector<int>& kv, int N, int nh, int nkv, int cap, int page, int window, int max_q) {
  return Batch{cu.data(), kv.data(), N, (int)kv.size(), (cap + page - 1) / page, page, window, nh, nkv, 64, max_q};
}

int main() {
  // offsets that go back: more items than workgroups, slots that nobody writes, unless nothing is computed
  {
    const std::vector<int> cu = {0, 400, 0, 400, 0, 368, 400}, kv = {0, 0, 0, 0, 0, 100000};
    const Batch b = batch(cu, kv, 400, 32, 8, 100000, 16, 0, 400);
    CHECK(chunk_list(b, false) > 0);
    CHECK(chunk_list(b, true) == 0);
  }
  {
    std::vector<int> cu(256), kv(255, 1024);
    for (int i = 0; i < 256; ++i) cu[i] = i % 2 ? 1024 : 0;
    kv[254] = 100000;
    const Batch b = batch(cu, kv, 1024, 1, 1, 100000, 16, 0, 1024);
    CHECK(chunk_list(b, false) > 0);
    CHECK(chunk_list(b, true) == 0);
  }
  std::mt19937 rng(11);
  auto below = [&](int n) { return n <= 0 ? 0 : (int)(rng() % (unsigned)n); };
  for (int round = 0; round < 3000; ++round) {
    const int R = 1 + below(round % 10 == 0 ? 700 : 40);
    const int N = 1 + below(round % 3 == 0 ? 60 : 5000);
    const int nkv = 1 << below(4), nh = nkv * (1 + below(8));
    std::vector<int> cu(R + 1), kv(R);
    const bool wild = round % 7 == 0;      // offsets outside the batch, lengths outside the table
    for (int& x : cu) x = wild ? below(2 * N) - N / 2 : below(N + 1);
    std::sort(cu.begin(), cu.end());
    const int cap = 1 << (4 + below(16));
    for (int& x : kv) x = wild ? (int)rng() : below(below(3) ? cap + 1 : 40);
    const Batch b = batch(cu, kv, N, nh, nkv, cap, 1 << below(8), below(2) ? 0 : 1 + below(3000), round % 2 ? N : 1 + below(3));
    if (count_items(b, kCus).chunks) CHECK(chunk_list(b, true) == 0);
    else few_list(b);
    Batch f = b;
    f.max_q = 1;                           // a hint that is too small selects the other list, with all rows
    if (!count_items(f, kCus).chunks) few_list(f);
  }
  // the longest requests that the arguments allow, many of them: no piece is lost to the limits of the piece sizes
  {
    std::vector<int> cu(1001), kv(1000, (1 << 30) - 1);
    for (int i = 0; i <= 1000; ++i) cu[i] = i;
    Batch b = batch(cu, kv, 1000, 8, 8, (1 << 30) - (1 << 20), 1 << 20, 0, 1);
    CHECK(count_items(b, kCus).chunks);
    CHECK(chunk_list(b, true) == 0);
    for (int i = 0; i <= 1000; ++i) cu[i] = 40 * i;
    b = batch(cu, kv, 40000, 8, 8, (1 << 30) - (1 << 20), 1 << 20, 0, 40);
    CHECK(chunk_list(b, true) == 0);
  }
  if (g_failed) return 1;
  std::puts("paged item checks passed");
  return 0;
}
