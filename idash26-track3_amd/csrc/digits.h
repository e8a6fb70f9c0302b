// digits.h -- ring words as balanced base-256 digits for the int8 matrix cores:
// device helpers of the ring products (gemm.hip, q4.hip, attn.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace mpcx {

typedef int v4i_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t ring_digits(uint32_t a) { return (a + 0x80808080u) ^ 0x80808080u; }

__device__ __forceinline__ uint64_t ring_digits64(uint64_t a) {
  return (a + 0x8080808080808080ull) ^ 0x8080808080808080ull;
}
// v_perm_b32 selector of output bytes j0..j0+3 for shift s: digit s - j (bytes
// 0..3 of the low source word, 4..7 of the high one), 0x0c (zero) when s < j
constexpr uint32_t digit_sel(int s, int j0) {
  uint32_t v = 0;
  for (int j = 0; j < 4; j++) v |= uint32_t(s - (j0 + j) >= 0 ? s - (j0 + j) : 0x0c) << (8 * j);
  return v;
}

// MFMA row operands of one 16-byte LDS read (16 Z_2^32 or 8 Z_2^64 words of a
// row, balanced digits): shift s takes digit s - j of each word at byte j
template <typename T>
__device__ __forceinline__ void digit_shifts(uint4 a, v4i_t (&as)[sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    constexpr uint32_t sel[4] = {0x0c0c0c00u, 0x0c0c0001u, 0x0c000102u, 0x00010203u};
#pragma unroll
    for (int q = 0; q < 4; q++)
      as[q] = v4i_t{int(__builtin_amdgcn_perm(0u, a.x, sel[q])), int(__builtin_amdgcn_perm(0u, a.y, sel[q])),
                    int(__builtin_amdgcn_perm(0u, a.z, sel[q])), int(__builtin_amdgcn_perm(0u, a.w, sel[q]))};
  } else {
#pragma unroll
    for (int q = 0; q < 8; q++) {
      const uint32_t lo = digit_sel(q, 0), hi = digit_sel(q, 4);
      as[q] = v4i_t{int(__builtin_amdgcn_perm(a.y, a.x, lo)), int(__builtin_amdgcn_perm(a.y, a.x, hi)),
                    int(__builtin_amdgcn_perm(a.w, a.z, lo)), int(__builtin_amdgcn_perm(a.w, a.z, hi))};
    }
  }
}
// digit_shifts for Z_2^32 with the byte selectors in scalar registers (set
// once per kernel by pan_shift_selectors): VOP3 takes no literal operand, so
// constant selectors are otherwise rematerialised in vector registers
struct ShiftSel {
  uint32_t s[4];
};
__device__ __forceinline__ ShiftSel pan_shift_selectors() {
  ShiftSel r;
  asm("s_mov_b32 %0, 0x0c0c0c00" : "=s"(r.s[0]));
  asm("s_mov_b32 %0, 0x0c0c0001" : "=s"(r.s[1]));
  asm("s_mov_b32 %0, 0x0c000102" : "=s"(r.s[2]));
  asm("s_mov_b32 %0, 0x00010203" : "=s"(r.s[3]));
  return r;
}
__device__ __forceinline__ void digit_shifts_s(uint4 a, const ShiftSel &sel, v4i_t (&as)[4]) {
#pragma unroll
  for (int q = 0; q < 4; q++)
    as[q] = v4i_t{int(__builtin_amdgcn_perm(0u, a.x, sel.s[q])), int(__builtin_amdgcn_perm(0u, a.y, sel.s[q])),
                  int(__builtin_amdgcn_perm(0u, a.z, sel.s[q])), int(__builtin_amdgcn_perm(0u, a.w, sel.s[q]))};
}
// the ring word of accumulator register r (shift sums acc[q][r])
template <typename T>
__device__ __forceinline__ T digit_fold(const v4i_t (&acc)[sizeof(T)], int r) {
  T v = 0;
#pragma unroll
  for (int q = 0; q < int(sizeof(T)); q++) {
    if constexpr (sizeof(T) == 4) v += uint32_t(acc[q][r]) << (8 * q);
    else v += uint64_t(int64_t(acc[q][r])) << (8 * q);
  }
  return v;
}

// Workgroup p of a one-dimensional launch of W runs on XCD p mod 8 (the
// dispatcher deals workgroups to the eight XCDs in turn); renumbering so that
// each XCD takes a contiguous range of W / 8 logical workgroups keeps a batch
// entry's tiles, which share their operands, in one XCD's L2.
constexpr int kXcds = 8;
__device__ __forceinline__ int xcd_swizzle(int p, int W) {
  const int xcd = p % kXcds, q = p / kXcds, base = W / kXcds, rem = W % kXcds;
  return (xcd < rem ? xcd * (base + 1) : rem * (base + 1) + (xcd - rem) * base) + q;
}

// balanced digits of a 16-byte group (four Z_2^32 words or two Z_2^64 words) of x - y
template <typename T>
__device__ __forceinline__ uint4 wide_digits(uint4 x, uint4 y) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(ring_digits(x.x - y.x), ring_digits(x.y - y.y), ring_digits(x.z - y.z), ring_digits(x.w - y.w));
  } else {
    const uint64_t lo = ring_digits64(((uint64_t(x.y) << 32) | x.x) - ((uint64_t(y.y) << 32) | y.x));
    const uint64_t hi = ring_digits64(((uint64_t(x.w) << 32) | x.z) - ((uint64_t(y.w) << 32) | y.z));
    return make_uint4(uint32_t(lo), uint32_t(lo >> 32), uint32_t(hi), uint32_t(hi >> 32));
  }
}

}  // namespace mpcx
