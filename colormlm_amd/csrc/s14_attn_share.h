// Do two packed [tokens][heads] operands, or one and a run of bytes, share memory?  Plain C++ (no HIP
// types): the library and a host-only test include it.
#pragma once

#include <cstdint>

namespace s14 {

// Rows of `row` bytes: (token t, head h) at address at + t * token + h * head.
struct RowBytes {
  uint64_t at, token, head, row;
  uint32_t heads;
  uint64_t bytes(uint32_t tokens) const { return uint64_t(tokens - 1) * token + uint64_t(heads - 1) * head + row; }
};

// Whether a row of a and a row of b have a byte in common, for `tokens` >= 1 of
// both.  own: a row of a may lie where the same row of b does.  Exact where
// both go from token to token, and from head to head, in the same steps, or have
// one of them: slices of one projection, whose extents always overlap.  Operands
// of other steps share memory where their extents do.
inline bool rows_share(const RowBytes &a, const RowBytes &b, uint32_t tokens, bool own) {
  if (a.at + a.bytes(tokens) <= b.at || b.at + b.bytes(tokens) <= a.at) return false;
  if ((tokens > 1 && a.token != b.token) || (a.heads > 1 && b.heads > 1 && a.head != b.head)) return true;
  const int64_t step = tokens > 1 ? int64_t(a.token) : 0, most = int64_t(tokens) - 1;
  const int64_t head = int64_t(a.heads > 1 ? a.head : b.head), from = int64_t(a.at - b.at);
  for (int64_t dh = -(int64_t(b.heads) - 1); dh < int64_t(a.heads); ++dh) {
    // rows of a and b that lie dh heads and dt tokens apart overlap where
    // -a.row < v + dt * step < b.row
    const int64_t v = from + dh * head, low = -int64_t(a.row) - v;
    int64_t dt = -most;
    if (step) {
      const int64_t down = low / step - (low % step < 0);  // floor
      if (down + 1 > dt) dt = down + 1;
    }
    for (; dt <= most; ++dt) {
      const int64_t d = v + dt * step;
      if (d >= int64_t(b.row)) break;
      if (d > -int64_t(a.row) && !(own && !dh && !dt && !from)) return true;
    }
  }
  return false;
}

// Whether one of `tokens` >= 1 rows of a, which has one head, and the `bytes` from
// address `from` have a byte in common.
inline bool rows_touch(const RowBytes &a, uint64_t from, uint64_t bytes, uint32_t tokens) {
  if (a.at + a.bytes(tokens) <= from || from + bytes <= a.at) return false;
  const uint64_t t = from < a.at + a.row ? 0 : (from - a.at - a.row) / a.token + 1;  // the first that ends past it
  return t < tokens && a.at + t * a.token < from + bytes;
}

}  // namespace s14
