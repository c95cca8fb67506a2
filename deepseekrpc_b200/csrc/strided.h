// Whether strided tensors meet in memory, found on the host before a launch.
#pragma once

#include <stdint.h>

#include <utility>

namespace dsr {

// The bytes base + i step[0] + j step[1] + [0, width) of i < count[0], j < count[1], in a
// normal form: steps positive, the larger first, adjacent pieces joined.
struct StridedBytes {
  using Wide = __int128;  // counts times steps of any 64-bit strides
  Wide base, width, step[2], end;  // end: behind the last byte
  int64_t count[2];

  StridedBytes() = default;
  StridedBytes(const void* p, int64_t width_, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int size)
      : base(reinterpret_cast<uintptr_t>(p)), width(Wide(width_) * size), step{Wide(s0) * size, Wide(s1) * size},
        count{n0, n1} {
    for (int d = 0; d < 2; ++d) {
      if (count[d] <= 1 || step[d] == 0) count[d] = 1, step[d] = 0;
      if (step[d] < 0) base += step[d] * (count[d] - 1), step[d] = -step[d];
    }
    if (step[0] < step[1]) std::swap(step[0], step[1]), std::swap(count[0], count[1]);
    if (step[1] == width && count[1] > 1) join(1);
    if (count[1] == 1 && step[0] == width && count[0] > 1) join(0);
    end = base + step[0] * (count[0] - 1) + step[1] * (count[1] - 1) + width;
  }
  void join(int d) { width *= count[d], count[d] = 1, step[d] = 0; }

  // Whether two of its own pieces meet.
  bool folds() const {
    for (int d = 0; d < 2; ++d)
      if (count[d] > 1 && step[d] < width) return true;
    if (count[0] == 1 || count[1] == 1 || step[0] >= step[1] * (count[1] - 1) + width) return false;
    // pieces i apart one way and j apart the other
    const int few = count[0] < count[1] ? 0 : 1;
    for (int64_t i = 1; i < count[few]; ++i) {
      const Wide at = step[few] * i, j = at / step[1 - few];
      for (Wide q = j; q <= j + 1; ++q)
        if (q >= 1 && q < count[1 - few] && at - q * step[1 - few] < width && q * step[1 - few] - at < width) return true;
    }
    return false;
  }

  // Whether a byte of both exists: b's place minus a's, a sum of steps times bounded whole
  // numbers, has to fall into a window.  The search takes the largest step first; with rows
  // that do not overlap each has one or two candidates.  Gives up (false) after kTries, as
  // only different strides over one another's memory need.
  static bool meet(const StridedBytes& a, const StridedBytes& b) {
    if (a.end <= b.base || b.end <= a.base) return false;
    Search s;
    for (int d = 0; d < 2; ++d) s.add(a.step[d], 1 - a.count[d], 0), s.add(b.step[d], 0, b.count[d] - 1);
    return s.find(0, a.base - b.base - b.width + 1, a.base - b.base + a.width - 1);
  }

 private:
  static Wide floor_div(Wide a, Wide b) { return a / b - (a % b < 0); }
  struct Search {
    static constexpr int kTries = 1 << 16;
    Wide step[4], low[4], high[4];
    int n = 0, tries = 0;
    void add(Wide s, Wide lo, Wide hi) {
      if (lo == hi) return;
      int at = 0;
      while (at < n && step[at] > s) ++at;
      if (at < n && step[at] == s) {
        low[at] += lo, high[at] += hi;
        return;
      }
      for (int i = n++; i > at; --i) step[i] = step[i - 1], low[i] = low[i - 1], high[i] = high[i - 1];
      step[at] = s, low[at] = lo, high[at] = hi;
    }
    bool find(int t, Wide from, Wide to) {  // a sum of the terms t.. in [from, to]
      if (t == n) return from <= 0 && 0 <= to;
      Wide least = 0, most = 0;
      for (int i = t + 1; i < n; ++i) least += step[i] * low[i], most += step[i] * high[i];
      Wide x = -floor_div(most - from, step[t]), last = floor_div(to - least, step[t]);
      if (x < low[t]) x = low[t];
      if (last > high[t]) last = high[t];
      for (; x <= last && tries < kTries; ++x) {
        ++tries;
        if (find(t + 1, from - x * step[t], to - x * step[t])) return true;
      }
      return false;
    }
  };
};

}  // namespace dsr
