// What the host checks of the operands of calls over packed sequences: their strides, and whether two share memory.
#pragma once
#include <stdint.h>

#include <numeric>

namespace qh {

constexpr int64_t kMaxStride = (int64_t)1 << 40;   // elements
constexpr int64_t kMaxSpan = (int64_t)1 << 61;     // bytes that a dimension may go over: every offset fits 64 bits

inline bool aligned_to_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// An operand [rows][heads][dim] with its element size, to check it and to compare it with another.
struct View {
  const void* p;
  int64_t rows, heads, dim, ld, hs;
  int eb;
  uintptr_t at() const { return reinterpret_cast<uintptr_t>(p); }
  int64_t width() const { return ((heads > 1 ? (heads - 1) * hs : 0) + dim) * eb; }             // bytes of a row's span
  int64_t bytes() const { return (rows > 1 ? (rows - 1) * ld * eb : 0) + width(); }
  // 16-byte pieces: pointer and strides (those of dimensions with one entry do not count)
  bool readable() const {
    return p && aligned_to_16(p) && (rows <= 1 || (ld >= 0 && ld < kMaxStride && ld * eb % 16 == 0)) &&
           (heads <= 1 || (hs >= 0 && hs < kMaxStride && hs * eb % 16 == 0));
  }
  // and width() and bytes() can be counted
  bool countable() const {
    auto span = [&](int64_t n, int64_t stride) { return n <= 1 || (__int128)(n - 1) * stride * eb <= kMaxSpan; };
    return span(rows, ld) && span(heads, hs) && span(2, dim);
  }
  // rows and heads any distance apart
  bool strided() const {
    return p && at() % eb == 0 && (rows <= 1 || (ld >= 0 && ld < kMaxStride)) && (heads <= 1 || (hs >= 0 && hs < kMaxStride));
  }
  // no two elements in one place
  bool writable() const { return readable() && distinct(); }
  bool distinct() const {
    if (rows > 1 && heads > 1)
      return hs >= dim && ld >= dim && ((__int128)(heads - 1) * hs <= ld - dim || (__int128)(rows - 1) * ld <= hs - dim);
    return (rows <= 1 || ld >= dim) && (heads <= 1 || hs >= dim);
  }
};

// One and the same operand.
inline bool same(const View& a, const View& b) {
  return a.p == b.p && a.rows == b.rows && a.heads == b.heads && a.dim == b.dim && a.eb == b.eb && (a.rows <= 1 || a.ld == b.ld) &&
         (a.heads <= 1 || a.hs == b.hs);
}
inline View flat(const void* p, int64_t n, int eb) { return {p, 1, 1, n, 0, 0, eb}; }

// Whether two operands (countable ones) share memory, as far as their spans and strides tell: they share none if the spans do
// not meet, or are disjoint columns of rows of one length, or if all their strides have a common divisor of which
// the one's pieces of `dim` elements and the other's take different parts (halves of each head, interleaved).
inline bool overlap(const View& a, const View& b) {
  if (a.at() >= b.at() + b.bytes() || b.at() >= a.at() + a.bytes()) return false;
  auto apart = [&](int64_t period, int64_t wa, int64_t wb) {
    if (wa > period || wb > period) return false;
    int64_t d = (int64_t)(b.at() - a.at()) % period;
    if (d < 0) d += period;
    return d >= wa && d + wb <= period;
  };
  if (a.rows > 1 && b.rows > 1 && a.ld * a.eb == b.ld * b.eb && a.ld > 0 && apart(a.ld * a.eb, a.width(), b.width())) return false;
  int64_t step = 0;
  for (const View* v : {&a, &b}) {
    if (v->rows > 1) step = std::gcd(step, v->ld * v->eb);
    if (v->heads > 1) step = std::gcd(step, v->hs * v->eb);
  }
  return !(step > 0 && apart(step, a.dim * a.eb, b.dim * b.eb));
}
template <class... V>
bool all_countable(const V&... v) {
  return (v.countable() && ...);
}
template <class... V>
bool overlap_any(const View& a, const V&... v) {
  return (overlap(a, v) || ...);
}

}  // namespace qh
