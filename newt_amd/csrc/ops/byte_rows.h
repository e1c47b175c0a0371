// Rows in memory, on the host.
#pragma once
#include <cstdint>

namespace newt_ops {

// Rows of `width` bytes, `stride` bytes apart.
struct ByteRows {
  int64_t first, rows, stride, width;
  ByteRows(const void* p, int64_t rows_, int64_t stride_, int64_t width_)
      : first((int64_t)(uintptr_t)p), rows(rows_), stride(rows_ > 1 ? stride_ : 0), width(width_) {
    if (stride < 0) {
      first += (rows - 1) * stride;
      stride = -stride;
    }
  }
  int64_t end() const { return first + (rows - 1) * stride + width; }
};

// Whether a byte of one lies in the other: a row at a time where all of them lie
// between each other's ends, as columns of one buffer do.
inline bool rows_meet(const ByteRows& a, const ByteRows& b) {
  if (a.rows <= 0 || b.rows <= 0 || a.first >= b.end() || b.first >= a.end()) return false;
  for (int64_t i = 0; i < a.rows; ++i) {
    // the last row of b that begins before this one of a ends
    const int64_t from = a.first + i * a.stride, before = from + a.width - 1 - b.first;
    if (before < 0) continue;
    int64_t j = b.stride ? before / b.stride : 0;
    if (j >= b.rows) j = b.rows - 1;
    if (b.first + j * b.stride + b.width > from) return true;
  }
  return false;
}

}  // namespace newt_ops
