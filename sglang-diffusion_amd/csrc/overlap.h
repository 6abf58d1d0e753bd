// Host checks of the rows that a call writes: whether they share memory with each other, or with rows that
// it reads.  Rows of a fused projection lie between each other's without touching, so spans alone do not
// tell.
#pragma once
#include <cstdint>
#include <cstdlib>
#include <utility>

namespace mi355 {

// n[0] * n[1] * n[2] rows of `width` bytes, s[] bytes apart in each direction.
struct Rows {
  const void* at;
  int64_t width;
  int64_t n[3], s[3];

  bool empty() const { return n[0] <= 0 || n[1] <= 0 || n[2] <= 0 || width <= 0; }
};

typedef __int128 wide_t;  // (2^31 rows, 2^41 bytes apart)

// Each row apart from the others.  Taken by their strides, smallest first, each direction has to step over
// all that the ones before it span.  (Rows that interleave in other ways are refused as well.)
inline bool rows_distinct(const Rows& r) {
  if (r.empty()) return true;
  wide_t span = r.width;
  bool done[3] = {r.n[0] == 1, r.n[1] == 1, r.n[2] == 1};
  for (;;) {
    int d = -1;
    for (int i = 0; i < 3; ++i)
      if (!done[i] && (d < 0 || std::abs(r.s[i]) < std::abs(r.s[d]))) d = i;
    if (d < 0) return true;
    if (std::abs(r.s[d]) < span) return false;
    span += (wide_t)(r.n[d] - 1) * std::abs(r.s[d]);
    done[d] = true;
  }
}

// The same rows, one by one.
inline bool rows_same(const Rows& a, const Rows& b) {
  bool same = a.at == b.at && a.width == b.width;
  for (int d = 0; d < 3; ++d) same = same && a.n[d] == b.n[d] && (a.n[d] <= 1 || a.s[d] == b.s[d]);
  return same;
}

// No row of a shares memory with one of b.  Exact where both have the same strides (a direction in which one
// of them has a single row takes the other's); with different ones, apart means that the spans are.
inline bool rows_apart(const Rows& a, const Rows& b) {
  if (a.empty() || b.empty()) return true;
  struct Span {
    wide_t lo, hi;
  };
  auto span = [](const Rows& r) {
    Span s{(wide_t)(uintptr_t)r.at, (wide_t)(uintptr_t)r.at + r.width};
    for (int d = 0; d < 3; ++d) (r.s[d] < 0 ? s.lo : s.hi) += (wide_t)(r.n[d] - 1) * r.s[d];
    return s;
  };
  const Span x = span(a), y = span(b);
  if (x.hi <= y.lo || y.hi <= x.lo) return true;
  // A row of b begins delta + sum of k[d] * s[d] behind one of a, k[d] the difference of their indices in
  // [lo, hi]: they meet if that can be in (-b.width, a.width).  Larger strides first: what the smaller ones
  // can add leaves a few k[d] each.
  struct Step {
    int64_t s, lo, hi;
  } step[3];
  for (int d = 0; d < 3; ++d) {
    if (a.n[d] > 1 && b.n[d] > 1 && a.s[d] != b.s[d]) return false;
    const int64_t s = a.n[d] > 1 ? a.s[d] : b.s[d];
    step[d] = s < 0 ? Step{-s, -(b.n[d] - 1), a.n[d] - 1} : Step{s, -(a.n[d] - 1), b.n[d] - 1};
  }
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if (step[j].s < step[j + 1].s) std::swap(step[j], step[j + 1]);
  int left = 4096;  // of combinations: beyond that they are taken to meet
  struct Search {
    const Step* step;
    wide_t below, above;  // what a difference has to be between
    int* left;
    bool meets(int d, wide_t delta) const {
      if (--*left < 0) return true;
      if (d == 3) return below < delta && delta < above;
      const Step& t = step[d];
      if (t.s == 0 || (t.lo == 0 && t.hi == 0)) return meets(d + 1, delta);
      wide_t least = 0, most = 0;  // of the directions behind this one
      for (int i = d + 1; i < 3; ++i) least += (wide_t)step[i].lo * step[i].s, most += (wide_t)step[i].hi * step[i].s;
      auto floor_div = [](wide_t p, wide_t q) { return p / q - (p % q < 0); };
      // below - most < delta + k s < above - least
      wide_t k = floor_div(below - most - delta, t.s) + 1;
      const wide_t end = -floor_div(-(above - least - delta), t.s) - 1;
      if (k < t.lo) k = t.lo;
      for (; k <= end && k <= t.hi; ++k)
        if (meets(d + 1, delta + k * t.s)) return true;
      return false;
    }
  };
  const Search search{step, -(wide_t)b.width, (wide_t)a.width, &left};
  return !search.meets(0, (wide_t)(uintptr_t)b.at - (wide_t)(uintptr_t)a.at);
}

}  // namespace mi355
