// overlap.h -- whether buffers of a call share bytes.  Plain C++, so that a program
// without a GPU can check it.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace mpcx {

// True where n1 bytes at p and n2 bytes at q do not overlap.
inline bool bytes_apart(const void *p, size_t n1, const void *q, size_t n2) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a + n1 <= b || b + n2 <= a;
}

// `rows` rows of `width` bytes, `pitch` (width or more) bytes apart.
struct ByteRows {
  const void *p;
  size_t rows, pitch, width;
  uintptr_t at() const { return reinterpret_cast<uintptr_t>(p); }
  bool none() const { return rows == 0 || width == 0; }
};
// True where no row has a byte of the n bytes at q.
inline bool rows_apart(const ByteRows &a, const void *q, size_t n) {
  if (a.none() || n == 0) return true;
  const uintptr_t p = a.at(), b = reinterpret_cast<uintptr_t>(q);
  const size_t i = b < p + a.width ? 0 : (b - (p + a.width)) / a.pitch + 1;  // the first row that ends past q
  return i >= a.rows || p + i * a.pitch >= b + n;
}
// True where the rows of a and b share no byte; a's may lie between b's (columns of one
// larger matrix).
inline bool rows_apart(const ByteRows &a, const ByteRows &b) {
  if (a.rows > b.rows) return rows_apart(b, a);
  if (a.none() || b.none()) return true;
  if (bytes_apart(a.p, (a.rows - 1) * a.pitch + a.width, b.p, (b.rows - 1) * b.pitch + b.width)) return true;
  if (a.pitch == b.pitch) {
    const uintptr_t p = a.at(), q = b.at();
    const size_t off = q >= p ? (q - p) % a.pitch : (a.pitch - (p - q) % a.pitch) % a.pitch;
    if (off >= a.width && off + b.width <= a.pitch) return true;
  }
  for (size_t i = 0; i < a.rows; i++)
    if (!rows_apart(b, reinterpret_cast<const void *>(a.at() + i * a.pitch), a.width)) return false;
  return true;
}

}  // namespace mpcx
