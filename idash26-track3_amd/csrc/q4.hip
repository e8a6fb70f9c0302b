// q4.hip -- masked activations times public 4-bit weights with group scales, on
// the int8 matrix cores.
//
// C[m, n] = sum_g scale[g, n] sum_{k in g} q[n, k] A[m, k] mod 2^bw.  A ring word
// is a sum of bw / 8 balanced digits, A = sum_p 2^(8p) d_p with d_p in [-128, 127],
// and a 4-bit weight shifted to the high half of a byte is the int8 16 q: one AND
// (the high halves of a word's bytes) or a shift and an AND (the low ones) turn 8
// packed weights into 8 operand bytes.  The digits of a word are rows of the MFMA's
// A operand: its 16 rows are the planes of 4 (Z_2^32) or 2 (Z_2^64) words m, the
// weights its one B operand, so nothing of the product is computed twice or dropped.
// Accumulator register r of lane (li, lg) is row 4 lg + r, column li: a lane holds
// four planes of one word, folds them, and multiplies by the group's scale.
// A chunk is S = 128, 64 or 32 k, the largest that divides the group; the sums of a
// chunk are at most 2^21, so the fold's shifts stay exact in 32 bits:
//   sum_p 2^(8p) a_p / 16 = (a_0 >> 4) + (a_1 << 4) + (a_2 << 12) + (a_3 << 20),
// in Z_2^64 with 64-bit sums of the pairs (a_0, a_1), (a_2, a_3), and the lanes of
// planes 4..7 (odd lg) shifted up by 32 at the end.
//
// What it costs: bw / 8 int8 multiply-adds a weight and word, half a byte a weight, a
// scale a group.  Few rows are bound by the weights' bytes and, below some 10 MB of
// them, by a launch's start; many by the matrix cores and, beside them, by the scales'
// multiply-adds, 5 vector instructions a chunk and tile.  The figures below are of one
// MI355X; "rows x K x N", groups of 128 unless said.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn.h"
#include "digits.h"
#include "launch_util.h"

namespace mpcx {
namespace {

template <typename T>
constexpr int kRows = 16 / int(sizeof(T));  // words m per MFMA tile

__device__ __forceinline__ v4i_t mfma64(v4i_t a, v4i_t b, v4i_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4i_t mfma32(long a, long b, v4i_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x32_i8(a, b, c, 0, 0, 0);
}

// Operand bytes of a chunk: S / 32 dwords of packed weights per lane (k = chunk S +
// (S / 4) lg + 8 d + 0..7 in dword d), as even and odd k: dwords lo(d), hi(d).
// A 64-k operand is lo(2o), lo(2o + 1), hi(2o), hi(2o + 1); a 32-k one lo(0), hi(0).
__device__ __forceinline__ uint32_t q4_lo(uint32_t w) { return (w << 4) & 0xf0f0f0f0u; }
__device__ __forceinline__ uint32_t q4_hi(uint32_t w) { return w & 0xf0f0f0f0u; }

// acc of one chunk: a, b are its S / 32 dword pairs (even k, odd k)
template <int S>
__device__ __forceinline__ v4i_t q4_product(const uint32_t (&ae)[S / 32], const uint32_t (&ao)[S / 32],
                                            const uint32_t (&be)[S / 32], const uint32_t (&bo)[S / 32]) {
  v4i_t acc = {0, 0, 0, 0};
  if constexpr (S == 32) {
    acc = mfma32(long(uint64_t(ae[0]) | uint64_t(ao[0]) << 32), long(uint64_t(be[0]) | uint64_t(bo[0]) << 32), acc);
  } else {
#pragma unroll
    for (int o = 0; o < S / 64; o++)
      acc = mfma64(v4i_t{int(ae[2 * o]), int(ae[2 * o + 1]), int(ao[2 * o]), int(ao[2 * o + 1])},
                   v4i_t{int(be[2 * o]), int(be[2 * o + 1]), int(bo[2 * o]), int(bo[2 * o + 1])}, acc);
  }
  return acc;
}
// The chunk's sum of the four planes of a lane, divided by 16, times the scale.
template <typename T>
__device__ __forceinline__ T q4_fold(v4i_t a, int32_t scale) {
  if constexpr (sizeof(T) == 4) {
    return (uint32_t(a[0] >> 4) + (uint32_t(a[1]) << 4) + (uint32_t(a[2]) << 12) + (uint32_t(a[3]) << 20)) *
           uint32_t(scale);
  } else {
    const int32_t t0 = (a[0] >> 4) + (a[1] << 4), t1 = (a[2] >> 4) + (a[3] << 4);
    return uint64_t(int64_t(t0) * scale) + (uint64_t(int64_t(t1) * scale) << 16);
  }
}

// eight words from p on, zero from the `have`-th on
template <typename T>
__device__ __forceinline__ void load8(const T *p, int have, bool vec, T (&w)[8]) {
  if (vec && have >= 8) {
    const uint4 *v = reinterpret_cast<const uint4 *>(p);
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; i++) {
      const uint4 x = v[i];
      __builtin_memcpy(&w[i * 16 / int(sizeof(T))], &x, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = i < have ? p[i] : T(0);
  }
}
// Plane p of eight words: the digits of the even and of the odd ones.
template <typename T>
__device__ __forceinline__ void plane8(const T (&w)[8], int p, uint32_t *even, uint32_t *odd) {
  uint32_t y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if constexpr (sizeof(T) == 4) {
      y[i] = w[i] + 0x80808080u;
    } else {
      const uint64_t v = w[i] + 0x8080808080808080ull;
      y[i] = p & 4 ? uint32_t(v >> 32) : uint32_t(v);
    }
  }
  const uint32_t b = uint32_t(p & 3), sel = b | (b + 4) << 8;
  auto four = [&](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(a3, a2, sel), __builtin_amdgcn_perm(a1, a0, sel), 0x05040100u) ^
           0x80808080u;
  };
  *even = four(y[0], y[2], y[4], y[6]);
  *odd = four(y[1], y[3], y[5], y[7]);
}

// ---------------------------------------------------------------------------
// Few rows: a workgroup takes 16 columns and MT MFMA tiles of rows; its (up to 16) waves
// take the chunks of K in turn and add up their sums through LDS, so that 4096 columns are
// 4096 waves, each with a few loads of the weights in flight.  DIRECT: a lane forms its
// digits from the words themselves (a word's planes are the rows li of its tile, so each
// word is taken apart once for every plane and column tile); else from the workspace.
// 1 x 4096 x 4096 in Z_2^32: 6.6 us, 9 MB of weights and scales at 1.4 TB/s, of which an
// empty kernel is 3; 5 x 8192 x 2047 in Z_2^64, groups of 64: 12.2 us and the digits' 4.8.
// ---------------------------------------------------------------------------
template <typename T, int S, int MT, bool DIRECT>
__global__ __launch_bounds__(1024) void k_q4_few(Q4Args<T> g, bool vec, int steps) {
  constexpr int R = kRows<T>, NP = int(sizeof(T)), ND = S / 32;
  __shared__ T red[16][MT][64];
  const int tid = int(threadIdx.x), lane = tid & 63, waves = int(blockDim.x) >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, lg = lane >> 4, p = li % NP;
  const int n = int(blockIdx.x) * 16 + li, nc = n < g.N ? n : g.N - 1;
  const int m0 = int(blockIdx.y) * MT * R;
  const uint32_t qrow = uint32_t(q4_row_bytes(g.K));
  const uint8_t *q = g.q + size_t(nc) * qrow;
  const int chunks = (g.K + S - 1) / S, per = g.group / S;
  T out[MT];
#pragma unroll
  for (int t = 0; t < MT; t++) out[t] = 0;
  const uint8_t *frag = static_cast<const uint8_t *>(g.work) + size_t(blockIdx.y) * MT * steps * 2048;
#pragma unroll 2
  for (int c = wave; c < chunks; c += waves) {
    const int kb = c * S + lg * (S / 4);  // this lane's first k
    uint32_t be[ND], bo[ND];
    // weights past the end of a row meet rows' zeros
    __builtin_memcpy(be, __builtin_assume_aligned(q + q4_place(qrow, S, c, lg), S / 8), 4 * ND);
    const int32_t scale = g.scale[size_t(c / per) * g.lds + nc];
#pragma unroll
    for (int d = 0; d < ND; d++) bo[d] = q4_hi(be[d]), be[d] = q4_lo(be[d]);
#pragma unroll
    for (int t = 0; t < MT; t++) {
      uint32_t ae[ND], ao[ND];
      if constexpr (DIRECT) {
        const int m = m0 + t * R + li / NP;
#pragma unroll
        for (int d = 0; d < ND; d++) {
          T w[8];
          load8<T>(g.a + size_t(m < g.M ? m : 0) * g.lda + kb + 8 * d, m < g.M ? g.K - kb - 8 * d : 0, vec, w);
          plane8<T>(w, p, &ae[d], &ao[d]);
        }
      } else {
        const uint8_t *f = frag + size_t(t) * steps * 2048 + size_t(c) * (16 * S);
        if constexpr (S == 32) {
          const uint2 v = reinterpret_cast<const uint2 *>(f)[lane];
          ae[0] = v.x, ao[0] = v.y;
        } else {
#pragma unroll
          for (int o = 0; o < ND / 2; o++) {
            const v4i_t v = reinterpret_cast<const v4i_t *>(f)[64 * o + lane];
            ae[2 * o] = v[0], ae[2 * o + 1] = v[1], ao[2 * o] = v[2], ao[2 * o + 1] = v[3];
          }
        }
      }
      out[t] += q4_fold<T>(q4_product<S>(ae, ao, be, bo), scale);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; t++) red[wave][t][lane] = out[t];
  __syncthreads();
  // word m of tile t, column li: lanes 16 lg.. (Z_2^64: 16 (2 lg).. and the planes above them)
  for (int e = tid; e < MT * R * 16; e += int(blockDim.x)) {
    const int t = e / (16 * R), r = e / 16 % R, col = e % 16;
    const int m = m0 + t * R + r, on = int(blockIdx.x) * 16 + col;
    T v = 0;
    for (int w = 0; w < waves; w++) {
      if constexpr (sizeof(T) == 4) v += red[w][t][16 * r + col];
      else v += red[w][t][32 * r + col] + (red[w][t][32 * r + 16 + col] << 32);
    }
    if (m < g.M && on < g.N) g.c[size_t(m) * g.ldc + on] = v;
  }
}

// ---------------------------------------------------------------------------
// Digits once for all columns, in the order the lanes take them.  The workspace holds,
// per MFMA tile of rows and step of 128 k, 2 KB of operands: 128 / S chunks of S / 64
// operands (64 lanes of 16 bytes; S = 32: one of 8 bytes).  768 x 4096 words of Z_2^32:
// 10.7 us, 25 MB in and out at 2.4 TB/s.
// ---------------------------------------------------------------------------
template <typename T, int S>
__global__ __launch_bounds__(256) void k_q4_digits(Q4Args<T> g, bool vec, int tiles, int steps, uint8_t *work) {
  constexpr int R = kRows<T>, NP = int(sizeof(T));
  const size_t per_row = size_t(steps) * 16, n = size_t(tiles) * R * per_row;  // groups of 8 words
  for (size_t e = size_t(blockIdx.x) * 256 + threadIdx.x; e < n; e += size_t(gridDim.x) * 256) {
    const int m = int(e / per_row), k = int(e % per_row) * 8;
    T w[8];
    load8<T>(g.a + size_t(m < g.M ? m : 0) * g.lda + k, m < g.M ? g.K - k : 0, vec, w);
    const int c = k / S, lg = k % S / (S / 4), d = k % (S / 4) / 8;
    uint8_t *tile = work + (size_t(m / R) * steps * (128 / S) + c) * (16 * S);
#pragma unroll
    for (int p = 0; p < NP; p++) {
      uint32_t even, odd;
      plane8<T>(w, p, &even, &odd);
      const int lane = 16 * lg + m % R * NP + p;
      if constexpr (S == 32) {
        *reinterpret_cast<uint2 *>(tile + 8 * lane) = make_uint2(even, odd);
      } else {
        uint32_t *o = reinterpret_cast<uint32_t *>(tile + (d / 2) * 1024 + 16 * lane);
        o[d % 2] = even;
        o[2 + d % 2] = odd;
      }
    }
  }
}

// Sums over chunks of plane sums times scales.  Z_2^32: one 24-bit multiply-add a plane
// (a chunk's plane sums are at most 2^21, divided by 16 in plane 0 so that no bit of the
// word is lost; the planes above need 4 fewer bits), the planes folded at the end; a
// scale past 24 bits is its low 12 bits and, in a second pass, the others.  Z_2^64:
// 64-bit sums of the plane pairs.
template <typename T>
struct Q4Sum;
template <>
struct Q4Sum<uint32_t> {
  uint32_t w[4];
  static __device__ __forceinline__ int32_t high(int32_t s) {
    return (uint32_t(s) + (1u << 23)) >> 24 ? s >> 12 : 0;
  }
  __device__ __forceinline__ void add(v4i_t a, int32_t s) {
    w[0] += uint32_t(__mul24(a[0] >> 4, s));
#pragma unroll
    for (int p = 1; p < 4; p++) w[p] += uint32_t(__mul24(a[p], s));
  }
  __device__ __forceinline__ void add_high(v4i_t a, int32_t s) {
#pragma unroll
    for (int p = 0; p < 4; p++) {
      int32_t x;  // (not __mul24, whose sign extensions would move to where every scale passes)
      asm("v_mul_i32_i24_e32 %0, %1, %2" : "=v"(x) : "v"(p ? a[p] : a[0] >> 4), "v"(s));
      w[p] += uint32_t(x) << 12;
    }
  }
  __device__ __forceinline__ uint32_t word() const {
    return w[0] + (w[1] << 4) + (w[2] << 12) + (w[3] << 20);
  }
};
template <>
struct Q4Sum<uint64_t> {
  uint64_t w[2];
  __device__ __forceinline__ void add(v4i_t a, int32_t s) {
    w[0] += uint64_t(int64_t((a[0] >> 4) + (a[1] << 4)) * s);
    w[1] += uint64_t(int64_t((a[2] >> 4) + (a[3] << 4)) * s);
  }
  static __device__ __forceinline__ int32_t high(int32_t) { return 0; }
  __device__ __forceinline__ void add_high(v4i_t, int32_t) {}
  __device__ __forceinline__ uint64_t word() const { return w[0] + (w[1] << 16); }
};

// Many rows: a workgroup of 2 x 2 waves, each MT tiles of rows by NT of columns.  The
// rows' operands of a step (128 k), which every column tile shares, go straight into LDS,
// the weights and scales, which only two waves share, to the lanes' registers (through
// LDS, too, they took as long); all are asked for a step ahead (two ahead: as long).  Two
// waves a SIMD (256 registers each), so that one's scales run beside the other's MFMAs.
// 768 x 4096 x 4096 in Z_2^32: 80.5 us, 1.28 POP/s of digits against 1.8 of a large int8
// product (Z_2^64: 163, 1.27): vector instructions issue 44% of the time and MFMAs 26%, each
// waiting for the other in a wave (all of a step's products in one block of code, the rare
// scales done over: 84), and 768 workgroups at two a CU are one and a half rounds.
template <typename T, int S, int MT, int NT>
__global__ __launch_bounds__(256, 2) void k_q4_many(Q4Args<T> g, int steps, const uint8_t *work) {
  constexpr int R = kRows<T>, ND = S / 32, CH = 128 / S;
  __shared__ __align__(16) v4i_t as0[2 * MT * 128], as1[2 * MT * 128];  // even and odd steps: tile, 2 KB
  const int gx = (g.N + 32 * NT - 1) / (32 * NT);
  const int lw = xcd_swizzle(int(blockIdx.x), int(gridDim.x));
  const int tid = int(threadIdx.x), lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = lw % gx * 32 * NT + (wave & 1) * 16 * NT, t0 = lw / gx * 2 * MT;
  const uint32_t qrow = uint32_t(q4_row_bytes(g.K));
  const int per = g.group / S, last = (g.K - 1) / S;
  // places in 32 bits from bases that a wave shares (launch_gemm_q4 bounds K)
  const int nw = min(n0, g.N - 1);
  const uint8_t *qw = g.q + size_t(nw) * qrow;
  const int32_t *sw = g.scale + nw;
  uint32_t qo[NT], so[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    so[t] = uint32_t(min(16 * t + li, g.N - 1 - nw));
    qo[t] = so[t] * qrow;
  }
  Q4Sum<T> out[MT][NT] = {};
  // 256 threads move two tiles of rows at a time
  const v4i_t *src = reinterpret_cast<const v4i_t *>(work) + size_t(t0) * steps * 128;
  const uint32_t ro = uint32_t(tid / 128 * steps * 128 + tid % 128);
  // a step's weights and scales
  struct Ahead {
    uint32_t b[CH][NT][ND];
    int32_t s[CH][NT];
  };
  auto load = [&](v4i_t *as, int step, Ahead &h) __attribute__((always_inline)) {
    step = min(step, steps - 1);
    // the rows' operands straight into LDS: a wave moves 64 groups of 16 bytes to
    // consecutive places
#pragma unroll
    for (int j = 0; j < MT; j++)
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void *)(src + (size_t(2 * j) * steps + step) * 128 + ro),
          (__attribute__((address_space(3))) void *)(as + 256 * j + 64 * wave), 16, 0, 0);
    // weights past the end of a row meet rows' zeros
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const int chunk = step * CH + c;
      const uint32_t at = q4_place(qrow, S, chunk, lg);
      const int32_t *sg = sw + size_t(min(chunk, last) / per) * g.lds;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        __builtin_memcpy(h.b[c][t], __builtin_assume_aligned(qw + (qo[t] + at), S / 8), 4 * ND);
        h.s[c][t] = sg[so[t]];
      }
    }
  };
  // Every wave's loads have landed, those into LDS (which the compiler does not wait for
  // at a barrier) among them, and the last step's operands are done with.
  auto arrived = [&](Ahead &h) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
      for (int t = 0; t < NT; t++) {  // here, so that their use does not wait for the loads that leave next
        asm volatile("" : "+v"(h.s[c][t]));
#pragma unroll
        for (int d = 0; d < ND; d++) asm volatile("" : "+v"(h.b[c][t][d]));
      }
  };
  auto compute = [&](const v4i_t *as, const Ahead &h) __attribute__((always_inline)) {
    const v4i_t *buf = as + (wave >> 1) * MT * 128;
#pragma unroll
    for (int c = 0; c < CH; c++) {
      uint32_t ae[MT][ND], ao[MT][ND];
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const v4i_t *a = buf + i * 128 + c * S;
        if constexpr (S == 32) {
          const uint2 v = reinterpret_cast<const uint2 *>(a)[lane];
          ae[i][0] = v.x, ao[i][0] = v.y;
        } else {
#pragma unroll
          for (int o = 0; o < ND / 2; o++) {
            const v4i_t v = a[64 * o + lane];
            ae[i][2 * o] = v[0], ae[i][2 * o + 1] = v[1], ao[i][2 * o] = v[2], ao[i][2 * o + 1] = v[3];
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        uint32_t be[ND], bo[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) be[d] = q4_lo(h.b[c][t][d]), bo[d] = q4_hi(h.b[c][t][d]);
        v4i_t acc[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) acc[i] = q4_product<S>(ae[i], ao[i], be, bo);
        const int32_t high = Q4Sum<T>::high(h.s[c][t]), low = h.s[c][t] - int32_t(uint32_t(high) << 12);
#pragma unroll
        for (int i = 0; i < MT; i++) out[i][t].add(acc[i], low);
        if (__any(high)) {
#pragma unroll
          for (int i = 0; i < MT; i++) out[i][t].add_high(acc[i], high);
        }
      }
    }
  };
  Ahead x, y;
  load(as0, 0, x);
  for (int step = 0; step < steps; step += 2) {
    arrived(x);
    load(as1, step + 1, y);
    compute(as0, x);
    if (step + 1 >= steps) break;
    arrived(y);
    load(as0, step + 2, x);
    compute(as1, y);
  }
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int n = n0 + 16 * t + li;
      T v = out[i][t].word();
      int r = lg;
      if constexpr (sizeof(T) == 8) {
        v += __shfl_xor(v, 16, 64) << 32;  // the planes above, from lane group lg + 1
        r = lg >> 1;
        if (lg & 1) continue;
      }
      const int m = (t0 + (wave >> 1) * MT + i) * R + r;
      if (m < g.M && n < g.N) g.c[size_t(m) * g.ldc + n] = v;
    }
}

constexpr int kManyMT = 4;
template <typename T>
int row_tiles(int M) {
  return (M + kRows<T> - 1) / kRows<T>;
}
// tiles in the workspace: whole workgroups of either kernel
template <typename T>
int work_tiles(int M) {
  return (row_tiles<T>(M) + 2 * kManyMT - 1) / (2 * kManyMT) * 2 * kManyMT;
}
int many_steps(int K) { return (K + 127) / 128; }
// Up to 16 tiles of rows take the first kernel.  4096 x 4096: 64 rows of Z_2^32 21.7 us,
// by the other 27.1; 128 rows 35.2, by the other 29.0; Z_2^64 in groups of 64: 32 rows
// 27.5, by the other 36.6; 64 rows 45.1, by the other 39.8.
constexpr int kFewTiles = 16;
template <typename T>
bool few_rows(int M) {
  return row_tiles<T>(M) <= kFewTiles;
}
// Its lanes form the digits themselves while that is little work, which the launch that
// forms them in the workspace costs more than.  Kernels, direct and with that launch:
// Z_2^32 32 x 1024 x 1024 5.5 us and 6.9, 1 x 4096 x 4096 6.6 and 7.7, at the line; 16 x
// 4096 x 4096 12.7 and 10.1, 1 x 8192 x 8192 20.1 and 17.0.  Z_2^64 1 x 2896 x 2880 7.3
// and 7.8, 4 x 2048 x 2048 7.6 and 8.1, at the line; 1 x 4096 x 4096 8.9 and 8.6, 4 x 4096
// x 4096 12.6 and 10.0.
template <typename T>
bool direct_rows(int M, int K, int N) {
  constexpr size_t most = size_t(sizeof(T) == 4 ? 1 << 20 : 1 << 19);  // words by column tile
  return few_rows<T>(M) && size_t(row_tiles<T>(M)) * K * ((size_t(N) + 15) / 16) <= most;
}

// launch(g) on as many columns at a time as `most` allows
template <typename T, class Fn>
hipError_t by_columns(const Q4Args<T> &g, size_t most, Fn &&launch) {
  for (size_t n = 0; n < size_t(g.N); n += most) {
    Q4Args<T> part = g;
    part.N = int(std::min(most, size_t(g.N) - n));
    part.q += n * q4_row_bytes(g.K);
    part.scale += n;
    part.c += n;
    const hipError_t e = launch(part);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int S>
hipError_t launch_at(const Launch &L, const Q4Args<T> &g) {
  const bool vec = reinterpret_cast<uintptr_t>(g.a) % 16 == 0 && g.lda % (16 / sizeof(T)) == 0;
  const bool direct = direct_rows<T>(g.M, g.K, g.N);
  const int tiles = work_tiles<T>(g.M), steps = many_steps(g.K);
  uint8_t *work = static_cast<uint8_t *>(g.work);
  if (!direct) {
    const size_t groups = size_t(tiles) * kRows<T> * steps * 16;
    const size_t want = (groups + 255) / 256, cap = size_t(L.num_cu) * 32;
    hipLaunchKernelGGL((k_q4_digits<T, S>), dim3(unsigned(want < cap ? want : cap)), dim3(256), 0, L.stream, g, vec, tiles,
                       steps, work);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (few_rows<T>(g.M)) {
    const int chunks = (g.K + S - 1) / S, waves = chunks < 16 ? chunks : 16;
    const int rt = row_tiles<T>(g.M);
    auto few = [&](auto mt) {
      constexpr int MT = decltype(mt)::value;
      return by_columns(g, kMostThreads / (64u * unsigned(waves)) * 16, [&](const Q4Args<T> &p) {
        const dim3 grid(unsigned((size_t(p.N) + 15) / 16), unsigned((rt + MT - 1) / MT)), block(64u * unsigned(waves));
        if (direct) hipLaunchKernelGGL((k_q4_few<T, S, MT, true>), grid, block, 0, L.stream, p, vec, steps);
        else hipLaunchKernelGGL((k_q4_few<T, S, MT, false>), grid, block, 0, L.stream, p, vec, steps);
        return hipGetLastError();
      });
    };
    if (rt >= 3) return few(std::integral_constant<int, 4>{});
    if (rt == 2) return few(std::integral_constant<int, 2>{});
    return few(std::integral_constant<int, 1>{});
  }
  const size_t rows = size_t(tiles / (2 * kManyMT)), enough = size_t(L.num_cu) * 2;
  auto many = [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    const size_t most = kMostThreads / 256 / rows;  // workgroups along the columns
    if (most == 0) return hipErrorInvalidValue;
    return by_columns(g, most * 32 * NT, [&](const Q4Args<T> &p) {
      const size_t wgs = (size_t(p.N) + 32 * NT - 1) / (32 * NT) * rows;
      hipLaunchKernelGGL((k_q4_many<T, S, kManyMT, NT>), dim3(unsigned(wgs)), dim3(256), 0, L.stream, p, steps, work);
      return hipGetLastError();
    });
  };
  // The widest column tiles that give every CU its two workgroups: 512 x 4096 x 4096 by 4
  // tiles 57.6 us, by 2 66.0; 256 rows by 4 40.0, by 2 35.8; 128 rows by 4 38.5, by 2 31.0,
  // by 1 28.1.  Groups of 32 hold twice the scales, too many for the registers of 4 tiles
  // (512 rows 438 us, by 2 161).
  auto wgs = [&](int nt) { return (size_t(g.N) + 32 * nt - 1) / (32 * nt) * rows; };
  if constexpr (S != 32)
    if (wgs(4) >= enough) return many(std::integral_constant<int, 4>{});
  if (wgs(2) >= enough) return many(std::integral_constant<int, 2>{});
  return many(std::integral_constant<int, 1>{});
}

}  // namespace

size_t q4_work_bytes(int bw, int M, int K) {
  return size_t(bw == 32 ? work_tiles<uint32_t>(M) : work_tiles<uint64_t>(M)) * many_steps(K) * 2048;
}

template <typename T>
hipError_t launch_gemm_q4(const Launch &L, const Q4Args<T> &g) {
  if (g.K > kQ4MaxK) return hipErrorInvalidValue;
  if (g.group % 128 == 0) return launch_at<T, 128>(L, g);
  if (g.group % 64 == 0) return launch_at<T, 64>(L, g);
  return launch_at<T, 32>(L, g);
}
template hipError_t launch_gemm_q4<uint32_t>(const Launch &, const Q4Args<uint32_t> &);
template hipError_t launch_gemm_q4<uint64_t>(const Launch &, const Q4Args<uint64_t> &);

}  // namespace mpcx
