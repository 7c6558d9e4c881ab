// Host checks of strided outputs: [tokens][heads] rows of `row` bytes each, any
// strides.  Two workgroups that write one element, or one that writes what
// another still reads, would leave what happens to come last.
#pragma once

#include <stdint.h>

namespace kvc {

struct RowSet {
  int64_t base, token, head;  // bytes
  int64_t tokens, heads;
};

inline RowSet row_set(const void* p, int64_t token_stride, int64_t head_stride, int64_t tokens, int64_t heads) {
  RowSet s = {static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)), tokens > 1 ? 2 * token_stride : 0, heads > 1 ? 2 * head_stride : 0,
              tokens, heads};
  if (s.token < 0) {
    s.base += (tokens - 1) * s.token;
    s.token = -s.token;
  }
  if (s.head < 0) {
    s.base += (heads - 1) * s.head;
    s.head = -s.head;
  }
  return s;
}

// Whether |x + t * step| < row for some |t| < count.
inline bool comes_near(int64_t x, int64_t step, int64_t count, int64_t row) {
  int64_t t = step ? -x / step : 0;  // the nearest are this one and its neighbours
  for (int64_t d = -1; d <= 1; ++d) {
    int64_t i = t + d;
    if (i > count - 1) i = count - 1;
    if (i < 1 - count) i = 1 - count;
    const int64_t y = x + i * step;
    if (y < row && -y < row) return true;
  }
  return false;
}

// Whether two rows of a set share bytes.
inline bool rows_share(const RowSet& s, int64_t row) {
  if (s.tokens < 1 || s.heads < 1) return false;
  if (s.tokens > 1 && s.token < row) return true;
  if (s.heads > 1 && s.head < row) return true;
  if (s.tokens == 1 || s.heads == 1) return false;
  const bool heads_near = s.head <= s.token;
  const int64_t near = heads_near ? s.head : s.token, near_count = heads_near ? s.heads : s.tokens;
  const int64_t far = heads_near ? s.token : s.head, far_count = heads_near ? s.tokens : s.heads;
  for (int64_t m = 1; m < far_count && m * far < near * (near_count - 1) + row; ++m)
    if (comes_near(m * far, near, near_count, row)) return true;
  return false;
}

// Whether rows of two sets of as many tokens share bytes.  Sets whose address
// ranges meet need the same token stride, and the same head stride unless they
// take turns as whole tokens: others are taken to share some.
inline bool rows_meet(const RowSet& a, const RowSet& b, int64_t row) {
  if (a.tokens < 1 || a.heads < 1 || b.heads < 1) return false;
  const int64_t tokens_a = (a.tokens - 1) * a.token, tokens_b = (b.tokens - 1) * b.token;
  const int64_t heads_a = (a.heads - 1) * a.head + row, heads_b = (b.heads - 1) * b.head + row;
  const int64_t apart = b.base - a.base;
  if (apart >= tokens_a + heads_a || -apart >= tokens_b + heads_b) return false;
  if (a.token != b.token) return true;
  if (a.token) {  // parts of the rows of one projection
    const int64_t at = (apart % a.token + a.token) % a.token;
    if (heads_a <= at && at + heads_b <= a.token) return false;
  }
  if (a.heads > 1 && b.heads > 1 && a.head != b.head) return true;
  const int64_t head = a.heads > 1 ? a.head : b.head;
  for (int64_t k = 1 - a.heads; k < b.heads; ++k)
    if (comes_near(apart + k * head, a.token, a.tokens, row)) return true;
  return false;
}

// `count` rows of `row` bytes, `step` apart; a vector is one row.
struct Rows {
  int64_t base, step, count, row;
};

inline Rows vector_rows(const void* p, int64_t bytes) {
  return {static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)), 0, p && bytes > 0 ? 1 : 0, bytes};
}

// Whether a vector and a set of rows in address order share bytes.
inline bool vector_meets(const Rows& v, const Rows& s) {
  if (v.count < 1 || s.count < 1 || s.row < 1 || v.base + v.row <= s.base) return false;
  const int64_t at = s.step > 0 && v.base > s.base ? (v.base - s.base) / s.step : 0;  // the last row that begins before it, or the first
  const int64_t first = at < s.count ? at : s.count - 1;
  if (v.base < s.base + first * s.step + s.row) return v.base + v.row > s.base + first * s.step;
  return first + 1 < s.count && v.base + v.row > s.base + (first + 1) * s.step;
}

}  // namespace kvc
