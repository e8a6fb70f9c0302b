// overlap.h -- whether rows that lie apart share bytes with another buffer.  Plain C++,
// so that a program without a GPU can check it.
#pragma once
#include <cstddef>
#include <cstdint>

namespace mpcx {

// `rows` rows of `width` bytes, `pitch` (width or more) bytes apart.
struct ByteRows {
  const void *p;
  size_t rows, pitch, width;
  uintptr_t at() const { return reinterpret_cast<uintptr_t>(p); }
  bool none() const { return rows == 0 || width == 0; }
  uintptr_t end() const { return at() + (rows - 1) * pitch + width; }
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
  if (a.end() <= b.at() || b.end() <= a.at()) return true;
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
