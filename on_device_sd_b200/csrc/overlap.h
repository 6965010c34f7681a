// Whether two strided tensors share memory, exactly: an operator whose output partly covers an input would read what it
// has already written.  Views of one buffer that interleave without touching (queries and keys of a fused projection, the two
// caches of one allocation) do not count.  Host only.
#pragma once
#include <cstdint>
#include <utility>

namespace b200moe {

// Rows of `width` bytes, which start at base + i0 * stride0 + i1 * stride1 + ... (bytes, strides not negative).
struct StridedRows {
  static constexpr int kMaxAxes = 3;
  uintptr_t base = 0;
  int64_t width = 0;
  int axes = 0;
  int64_t count[kMaxAxes] = {}, stride[kMaxAxes] = {};

  void axis(int64_t n, int64_t s) {
    count[axes] = n;
    stride[axes++] = n > 1 ? s : 0;
  }
  bool empty() const {
    for (int i = 0; i < axes; ++i)
      if (count[i] <= 0) return true;
    return width <= 0;
  }
  bool same(const StridedRows& o) const {
    if (base != o.base || width != o.width || axes != o.axes) return false;
    for (int i = 0; i < axes; ++i)
      if (count[i] != o.count[i] || stride[i] != o.stride[i]) return false;
    return true;
  }
};

namespace overlap_detail {
// One unknown per axis: lo <= x <= hi, worth s * x bytes.  Looks for values with near < c + sum s * x < far.
struct Unknowns {
  int n = 0;
  int64_t s[2 * StridedRows::kMaxAxes], lo[2 * StridedRows::kMaxAxes], hi[2 * StridedRows::kMaxAxes];
  int64_t rest_lo[2 * StridedRows::kMaxAxes + 1], rest_hi[2 * StridedRows::kMaxAxes + 1];   // what the unknowns from k on can add
  int64_t steps = 0;
};
inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }   // b > 0
constexpr int64_t kMaxSteps = 1 << 22;
inline bool reachable(Unknowns& u, int k, int64_t c, int64_t near, int64_t far) {
  if (c + u.rest_hi[k] <= near || c + u.rest_lo[k] >= far) return false;
  if (k == u.n) return true;
  const int64_t first = -floor_div(c + u.rest_hi[k + 1] - near - 1, u.s[k]), last = floor_div(far - 1 - c - u.rest_lo[k + 1], u.s[k]);
  for (int64_t x = first > u.lo[k] ? first : u.lo[k]; x <= u.hi[k] && x <= last; ++x) {
    if (++u.steps > kMaxSteps) return true;       // rows that cross each other that often: not told apart any further
    if (reachable(u, k + 1, c + u.s[k] * x, near, far)) return true;
  }
  return false;
}
}  // namespace overlap_detail

inline bool rows_meet(const StridedRows& a, const StridedRows& b) {
  if (a.empty() || b.empty()) return false;
  overlap_detail::Unknowns u;
  auto add = [&u](int64_t s, int64_t lo, int64_t hi) {
    if (s == 0 || lo == hi) return;
    for (int i = 0; i < u.n; ++i)
      if (u.s[i] == s) {            // the same stride in both: only the difference counts
        u.lo[i] += lo;
        u.hi[i] += hi;
        return;
      }
    u.s[u.n] = s; u.lo[u.n] = lo; u.hi[u.n++] = hi;
  };
  for (int i = 0; i < a.axes; ++i) add(a.stride[i], 0, a.count[i] - 1);
  for (int i = 0; i < b.axes; ++i) add(b.stride[i], 1 - b.count[i], 0);
  for (int i = 1; i < u.n; ++i)     // widest stride first: it leaves the fewest values
    for (int j = i; j > 0 && u.s[j] > u.s[j - 1]; --j) {
      std::swap(u.s[j], u.s[j - 1]);
      std::swap(u.lo[j], u.lo[j - 1]);
      std::swap(u.hi[j], u.hi[j - 1]);
    }
  u.rest_lo[u.n] = u.rest_hi[u.n] = 0;
  for (int i = u.n - 1; i >= 0; --i) {
    u.rest_lo[i] = u.rest_lo[i + 1] + u.s[i] * u.lo[i];
    u.rest_hi[i] = u.rest_hi[i + 1] + u.s[i] * u.hi[i];
  }
  // a row of a begins at d from a row of b: they share a byte when -a.width < d < b.width
  return overlap_detail::reachable(u, 0, (int64_t)a.base - (int64_t)b.base, -a.width, b.width);
}

}  // namespace b200moe
