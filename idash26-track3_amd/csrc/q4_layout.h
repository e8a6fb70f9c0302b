// q4_layout.h -- places in a row of packed 4-bit weights.  Plain C++, so that a
// program without a GPU can check them.
#pragma once
#include <cstddef>
#include <cstdint>

namespace mpcx {

// bytes of a row of K weights, two a byte, in whole 16
constexpr size_t q4_row_bytes(int K) { return (size_t(K) + 31) / 32 * 16; }

// Byte of a row of `row` bytes from which lane group lg takes its S / 8 bytes (S / 4
// weights) of chunk c.  Past the row's end they are the row's last bytes: a chunk may be
// longer than the row, and a lane group's place in it outside, and what is read there
// meets the operand's zeros.
constexpr uint32_t q4_place(uint32_t row, int S, int c, int lg) {
  const uint32_t at = uint32_t(c) * uint32_t(S / 2) + uint32_t(lg) * uint32_t(S / 8), end = row - uint32_t(S / 8);
  return at < end ? at : end;
}

}  // namespace mpcx
