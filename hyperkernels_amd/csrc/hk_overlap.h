// hk_overlap.h - whether the memory of two strided tensors meets, for the host's checks of outputs. Every workgroup of a
// launch may read and write at any time, so an output may lie on an input only where the same element of both is
// the same memory, and nowhere on another output.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace hk {

// Rows of `width` bytes, n[i] of them `step[i]` bytes apart in each of up to three directions. Directions of one
// row, or of rows that are the same memory (step 0), are left out; steps are positive, falling.
struct Rows {
  int64_t lo = 0, width = 0;  // first byte; width 0: no memory
  int dims = 0;
  int64_t n[3], step[3];
  int given = 0;  // directions as they were given, left out or not
  int64_t given_n[3], given_step[3];
  bool repeats = false;  // a direction of more than one row had step 0

  Rows(const void* p, int64_t elem, int64_t cols) : lo(reinterpret_cast<intptr_t>(p)), width(p ? elem * cols : 0) {}
  Rows& along(int64_t count, int64_t bytes) {
    if (count <= 0) width = 0;
    given_n[given] = count, given_step[given++] = count > 1 ? bytes : 0;
    if (count <= 1 || width == 0) return *this;
    if (bytes == 0) {
      repeats = true;
      return *this;
    }
    if (bytes < 0) lo += (count - 1) * bytes, bytes = -bytes;
    int i = dims++;
    for (; i > 0 && step[i - 1] < bytes; --i) n[i] = n[i - 1], step[i] = step[i - 1];
    n[i] = count, step[i] = bytes;
    return *this;
  }
  int64_t extent() const {
    int64_t e = width;
    for (int i = 0; i < dims; ++i) e += (n[i] - 1) * step[i];
    return e;
  }
  // The same memory for the same element.
  bool same(const Rows& o) const {
    if (lo != o.lo || width != o.width || given != o.given || repeats || o.repeats) return false;
    for (int i = 0; i < given; ++i)
      if (given_n[i] != o.given_n[i] || given_step[i] != o.given_step[i]) return false;
    return true;
  }
};

namespace detail {
// The rows of two tensors by their common directions: na and nb rows, 1 where a tensor has none there. a_rest and
// b_rest: the extents of what lies behind a direction.
struct Meeting {
  int dims = 0;
  int64_t na[6], nb[6], step[6], a_rest[6], b_rest[6];
  int64_t a_width, b_width;
  int budget = 4096;  // of steps; a search that needs more has no answer

  // Whether a row of b, `apart` bytes behind a row of a, meets it for some choice of rows in the directions from i
  // on. moved: not the same row; where it is false that one does not count.
  bool search(int i, int64_t apart, bool moved) {
    if (--budget < 0) return true;
    if (i == dims) return moved && apart < a_width && -apart < b_width;
    // k rows further: apart + k step has to lie within (-b_rest, a_rest)
    const int64_t lo = std::max(-(na[i] - 1), floor_div(-b_rest[i] - apart, step[i]) + 1);
    const int64_t hi = std::min(nb[i] - 1, -floor_div(apart - a_rest[i], step[i]) - 1);
    for (int64_t k = lo; k <= hi; ++k)
      if (search(i + 1, apart + k * step[i], moved || k != 0)) return true;
    return false;
  }
  static int64_t floor_div(int64_t x, int64_t y) { return x / y - (x % y < 0 ? 1 : 0); }
};
inline Meeting make_meeting(const Rows& a, const Rows& b) {
  Meeting m;
  m.a_width = a.width, m.b_width = b.width;
  for (int i = 0, j = 0; i < a.dims || j < b.dims; ++m.dims) {
    const int64_t sa = i < a.dims ? a.step[i] : 0, sb = j < b.dims ? b.step[j] : 0;
    m.step[m.dims] = std::max(sa, sb);
    m.na[m.dims] = sa >= sb ? a.n[i++] : 1;
    m.nb[m.dims] = sb >= sa ? b.n[j++] : 1;
  }
  int64_t ra = a.width, rb = b.width;
  for (int i = m.dims - 1; i >= 0; --i) {
    m.a_rest[i] = ra, m.b_rest[i] = rb;
    ra += (m.na[i] - 1) * m.step[i];
    rb += (m.nb[i] - 1) * m.step[i];
  }
  return m;
}
}  // namespace detail

// Whether some row of a and some row of b share memory. Exact, but for layouts whose rows interleave in ways that no
// view of a tensor has: there it may say so of two that do not.
inline bool overlap(const Rows& a, const Rows& b) {
  if (a.width == 0 || b.width == 0 || a.lo >= b.lo + b.extent() || b.lo >= a.lo + a.extent()) return false;
  return detail::make_meeting(a, b).search(0, b.lo - a.lo, true);
}
// Whether an output lies on what another workgroup reads: not where both are the same memory element by element.
inline bool overlap_unless_same(const Rows& out, const Rows& in) { return !out.same(in) && overlap(out, in); }
// Whether two rows of one output share memory.
inline bool overlaps_itself(const Rows& a) {
  if (a.width == 0) return false;
  return a.repeats || detail::make_meeting(a, a).search(0, 0, false);
}

}  // namespace hk
