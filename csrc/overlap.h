// Whether two strided blocks of memory share a byte. Plain C++, so it builds with g++ as well.
#pragma once
#include <algorithm>
#include <cstdint>
#include <utility>

namespace dpa {

// Bytes start + sum_i j_i stride_i, 0 <= j_i < size_i: dimensions with the larger strides first, those of one entry or
// stride 0 left out, neighbours that run on into each other joined. The last has stride 1: the bytes of an element.
struct Block {
  static constexpr int kMaxDims = 8;
  int64_t start = 0;
  int n = 0;
  bool empty = false;
  int64_t size[kMaxDims], stride[kMaxDims];

  template <class Sizes, class Strides>
  Block(const void* p, const Sizes& sizes, const Strides& strides, int dims, int64_t elem) : start((int64_t)(uintptr_t)p) {
    std::pair<int64_t, int64_t> d[kMaxDims];
    int m = 0;
    for (int i = 0; i < dims; ++i) {
      if (sizes[i] == 0) empty = true;
      if (sizes[i] > 1 && strides[i] != 0) d[m++] = {strides[i] * elem, sizes[i]};
    }
    d[m++] = {1, elem};
    std::sort(d, d + m, [](const auto& x, const auto& y) { return x.first > y.first; });
    for (int i = 0; i < m; ++i) {
      if (n > 0 && stride[n - 1] == d[i].first * d[i].second) {
        size[n - 1] *= d[i].second;
        stride[n - 1] = d[i].first;
      } else {
        size[n] = d[i].second;
        stride[n++] = d[i].first;
      }
    }
  }
  // bytes from the first to the last of dimensions i and up
  int64_t extent(int i) const {
    int64_t e = 1;
    for (; i < n; ++i) e += (size[i] - 1) * stride[i];
    return e;
  }
};

enum class Share { kApart, kOverlap, kUnknown };

// Dimensions j of b and up, beginning at byte d, and the run of bytes [0, len). Of b's rows that reach into the run, all but
// the first and the last lie inside it.
inline bool run_share(int64_t len, const Block& b, int j, int64_t d) {
  const int64_t e = b.extent(j);
  if (d >= len || d + e <= 0) return false;
  if (d >= 0 || d + e <= len || j == b.n - 1) return true;      // (b's first or last byte is one of its own)
  const int64_t s = b.stride[j], inner = b.extent(j + 1);
  const int64_t first = d + inner > 0 ? 0 : (-d - inner) / s + 1, last = std::min(b.size[j] - 1, (len - 1 - d) / s);
  if (last - first > 1 && inner <= s) return true;
  for (int64_t r = first; r <= last; ++r)
    if (run_share(len, b, j + 1, d + r * s)) return true;
  return false;
}

// Dimensions i of a and j of b and up, b beginning d bytes behind a. With a common outer stride s, and inner parts that fit
// into it, d = t s + e leaves two inner offsets, e in [0, s) and e - s, each possible if some pair of rows is t (t + 1)
// apart. kUnknown: strides that do not fit together.
inline Share share(const Block& a, int i, const Block& b, int j, int64_t d) {
  if (d >= a.extent(i) || -d >= b.extent(j)) return Share::kApart;
  if (i == a.n - 1) return run_share(a.size[i], b, j, d) ? Share::kOverlap : Share::kApart;
  if (j == b.n - 1) return run_share(b.size[j], a, i, -d) ? Share::kOverlap : Share::kApart;
  const int64_t s = std::max(a.stride[i], b.stride[j]);
  const bool ra = a.stride[i] == s, rb = b.stride[j] == s;
  const int64_t na = ra ? a.size[i] : 1, nb = rb ? b.size[j] : 1;
  const int ia = ra ? i + 1 : i, jb = rb ? j + 1 : j;
  if (a.extent(ia) > s || b.extent(jb) > s) return Share::kUnknown;
  const int64_t t = d >= 0 ? d / s : -((-d + s - 1) / s), e = d - t * s;
  Share all = Share::kApart;
  for (int k = 0; k < 2; ++k) {
    const int64_t rows = t + k;                     // a's row less b's
    if (rows > na - 1 || rows < -(nb - 1)) continue;
    const Share one = share(a, ia, b, jb, e - k * s);
    if (one == Share::kOverlap) return one;
    if (one == Share::kUnknown) all = one;
  }
  return all;
}
inline Share share(const Block& a, const Block& b) {
  if (a.empty || b.empty) return Share::kApart;
  return share(a, 0, b, 0, b.start - a.start);
}

}  // namespace dpa
