// csrc/overlap.h against sets of bytes, built by tests/test_overlap_cpu.py with g++ under AddressSanitizer + UBSan.
#include <cstdio>
#include <random>
#include <set>
#include <vector>

#include "overlap.h"

using dpa::Block;
using dpa::Share;

typedef std::vector<int64_t> Ints;
static std::set<int64_t> bytes(int64_t start, const Ints& sizes, const Ints& strides, int64_t elem) {
  std::set<int64_t> at = {start};
  for (size_t i = 0; i < sizes.size(); ++i) {
    std::set<int64_t> next;
    for (int64_t x : at)
      for (int64_t j = 0; j < sizes[i]; ++j) next.insert(x + j * strides[i] * elem);
    at = next;
  }
  std::set<int64_t> all;
  for (int64_t x : at)
    for (int64_t j = 0; j < elem; ++j) all.insert(x + j);
  return all;
}

static int g_failed = 0, g_unknown = 0, g_overlap = 0, g_apart = 0;
static void check(int64_t p, const Ints& sa, const Ints& ta, int64_t q, const Ints& sb, const Ints& tb, int64_t elem, bool known) {
  const Block a((const void*)p, sa, ta, (int)sa.size(), elem), b((const void*)q, sb, tb, (int)sb.size(), elem);
  const auto x = bytes(p, sa, ta, elem), y = bytes(q, sb, tb, elem);
  bool both = false;
  for (int64_t v : y) both |= x.count(v) > 0;
  for (int turn = 0; turn < 2; ++turn) {
    const Share s = turn ? share(b, a) : share(a, b);
    if (s == Share::kUnknown) {
      ++g_unknown;
      if (known) ++g_failed;
    } else {
      ++(both ? g_overlap : g_apart);
      if ((s == Share::kOverlap) != both) {
        ++g_failed;
        std::fprintf(stderr, "wrong: sizes %zu, offset %lld: %d\n", sa.size(), (long long)(q - p), (int)both);
      }
    }
  }
}

int main() {
  std::mt19937 rng(3);
  auto below = [&](int n) { return (int64_t)(rng() % (unsigned)n); };
  for (int round = 0; round < 20000; ++round) {
    const int64_t elem = int64_t(1) << below(3);
    // two slices of one dense block [s0, s1, s2, s3], possibly with its dimensions in another order
    const Ints full = {1 + below(4), 1 + below(4), 1 + below(4), 1 + below(5)};
    const Ints st = {full[1] * full[2] * full[3], full[2] * full[3], full[3], 1};
    Ints sa(4), sb(4);
    int64_t pa = 4096, pb = 4096;
    for (int i = 0; i < 4; ++i) {
      const int64_t la = below((int)full[i]), lb = below((int)full[i]);
      sa[i] = 1 + below((int)(full[i] - la));
      sb[i] = 1 + below((int)(full[i] - lb));
      pa += la * st[i] * elem;
      pb += lb * st[i] * elem;
    }
    check(pa, sa, st, pb, sb, st, elem, false);
    Ints order = {0, 1, 2, 3};
    std::shuffle(order.begin(), order.end(), rng);
    Ints sp, tp;
    for (int64_t i : order) {
      sp.push_back(sa[i]);
      tp.push_back(st[i]);
    }
    check(pa, sp, tp, pb, sb, st, elem, false);
    // unrelated strides, from any place
    const Ints sx = {1 + below(3), 1 + below(6)}, sy = {1 + below(3), 1 + below(6)};
    check(64 + below(40) * elem, sx, {below(12), 1}, 64 + below(40) * elem, sy, {below(12), 1}, elem, false);
  }
  // the layouts in use: columns of a fused projection, keys and values side by side in a page, a row or a head at a time
  check(0, {5, 3, 8}, {48, 8, 1}, 24 * 2, {5, 3, 8}, {48, 8, 1}, 2, true);
  check(0, {5, 3, 8}, {48, 8, 1}, 8 * 2, {5, 3, 8}, {48, 8, 1}, 2, true);
  check(0, {4, 6, 2, 8}, {192, 16, 8, 1}, 96 * 2, {4, 6, 2, 8}, {192, 16, 8, 1}, 2, true);
  check(0, {4, 6, 2, 8}, {192, 32, 8, 1}, 16 * 2, {4, 6, 2, 8}, {192, 32, 8, 1}, 2, true);
  check(0, {4, 6, 2, 8}, {96, 8, 48, 1}, 0, {1, 2, 8}, {16, 8, 1}, 2, true);
  check(0, {4, 100}, {103, 1}, 4, {4, 100}, {103, 1}, 4, true);
  std::printf("%d overlap, %d apart, %d unknown, %d wrong\n", g_overlap, g_apart, g_unknown, g_failed);
  if (g_failed || g_unknown * 5 > g_overlap + g_apart) return 1;
  std::puts("overlap checks passed");
  return 0;
}
