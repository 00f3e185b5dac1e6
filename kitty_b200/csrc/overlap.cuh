// Whether an output of a call shares memory with its inputs or with another output (host only).
//
// A tensor of a call is rows of `run` bytes at `at` + sum(i * step), 0 <= i < size.  Two of them meet where the distance of
// their bases plus sum(k * step) comes closer to zero than a row is long, k from -(size - 1) to 0 for the steps of the
// first, 0 to size - 1 for those of the second (equal steps add up).  From the largest step down only those k are
// looked at that the smaller steps can still make up for: two or three a step where steps nest, as those of views of one buffer
// do.  Tensors whose spans are apart, which is the rule, take a few comparisons.
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace kitty {

struct Rows {
  const void *at;
  int64_t size[3], step[3];      // steps in bytes
  int64_t run;
};

struct RowSteps {
  int n;
  int64_t step[6], lo[6], hi[6], least[7], most[7];      // ascending; least / most: what the steps below add up to
  int64_t run;
  int left;                                              // steps that do not nest: rather refused than looked at for long

  bool reach(int i, int64_t at) {
    if (--left < 0) return true;
    if (i < 0) return at < run && -at < run;
    auto down = [](int64_t x, int64_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
    int64_t first = -down(run - 1 + most[i] + at, step[i]), last = down(run - 1 - least[i] - at, step[i]);
    if (first < lo[i]) first = lo[i];
    if (last > hi[i]) last = hi[i];
    for (int64_t k = first; k <= last; ++k)
      if (reach(i - 1, at + k * step[i])) return true;
    return false;
  }
};

inline bool rows_meet(Rows x, Rows y) {
  int64_t end[2];
  for (Rows *r : {&x, &y}) {
    int64_t &e = end[r == &y];
    e = r->run;
    for (int i = 0; i < 3; ++i) {
      if (r->size[i] < 1) return false;
      if (r->step[i] < 0) {                              // the same rows from the other end
        r->at = static_cast<const char *>(r->at) + (r->size[i] - 1) * r->step[i];
        r->step[i] = -r->step[i];
      }
      e += (r->size[i] - 1) * r->step[i];
    }
  }
  const int64_t gap = static_cast<int64_t>(reinterpret_cast<uintptr_t>(y.at)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(x.at));
  if (gap >= end[0] || -gap >= end[1]) return false;
  RowSteps s{};
  for (int which = 0; which < 2; ++which)
    for (int d = 0; d < 3; ++d) {
      const int64_t size = which ? y.size[d] : x.size[d], step = which ? y.step[d] : x.step[d];
      if (size == 1 || step == 0) continue;
      int i = 0;
      while (i < s.n && s.step[i] < step) ++i;
      if (i == s.n || s.step[i] != step) {
        for (int j = s.n++; j > i; --j) s.step[j] = s.step[j - 1], s.lo[j] = s.lo[j - 1], s.hi[j] = s.hi[j - 1];
        s.step[i] = step;
        s.lo[i] = s.hi[i] = 0;
      }
      (which ? s.hi[i] : s.lo[i]) += which ? size - 1 : 1 - size;
    }
  for (int i = 0; i < s.n; ++i) {
    s.least[i + 1] = s.least[i] + s.lo[i] * s.step[i];
    s.most[i + 1] = s.most[i] + s.hi[i] * s.step[i];
  }
  s.run = x.run;                                         // rows of one call are of one length
  s.left = 20000;
  return s.reach(s.n - 1, gap);
}

inline bool same_rows(const Rows &x, const Rows &y) {
  if (x.at != y.at || x.run != y.run) return false;
  for (int i = 0; i < 3; ++i)
    if (x.size[i] != y.size[i] || (x.size[i] > 1 && x.step[i] != y.step[i])) return false;
  return true;
}

}  // namespace kitty
