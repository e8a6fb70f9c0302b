// q8.hip -- masked activations times public 8-bit weights, with a scale for each output
// channel and each token, on the int8 matrix cores.
//
// C[m, n] = tok[m] scale[n] sum_k q[n, k] A[m, k] mod 2^bw.  A ring word is a sum of
// bw / 8 balanced digits, A = sum_p 2^(8p) d_p with d_p in [-128, 127], and a weight is one
// int8, so a word takes bw / 8 digit products (planes) with the weights as they lie in
// memory: a lane's 16 bytes of a row are an MFMA's operand.  A plane's sum over k is at
// most 2^14 a term: 2^16 terms stay within 31 bits.  In Z_2^32 a sum that wraps would not
// matter, in Z_2^64 it would, so nobody sums more than 2^16 terms in 32 bits.
// The scales are multiplied at the end, once a word.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn.h"
#include "digits.h"
#include "launch_util.h"

namespace mpcx {
namespace {

constexpr int kExact = 1 << 16;  // terms of a 32-bit plane sum
constexpr int kRsrcWord3 = 0x00020000;  // buffer resource: 32-bit offsets

__device__ __forceinline__ v4i_t mfma64(v4i_t a, v4i_t b, v4i_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// Four words of a row from k on, zero from K on: the row's last four, moved down.  Without a
// branch a lane: at a join the compiler waits for the loads before it, group after group.
template <typename T>
struct Four {
  T w[4];
  __device__ __forceinline__ void load(const T *row, int k, int K) {
    if (K >= 4) {
      __builtin_memcpy(w, row + min(k, K - 4), sizeof w);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = row[min(i, K - 1)];
    }
  }
  __device__ __forceinline__ void cut(int k, int K) {
    const int down = K >= 4 ? max(k - (K - 4), 0) : 0, have = K - k;
    if (down & 1) w[0] = w[1], w[1] = w[2], w[2] = w[3];
    if (down & 2) w[0] = w[2], w[1] = w[3];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = i < have ? w[i] : T(0);
  }
};
// Bytes 0..3 of four 32-bit words, each byte's four side by side: with the words offset by
// 0x80 a byte, the digits.
__device__ __forceinline__ void bytes4(const uint32_t (&y)[4], uint32_t *d) {
  const uint32_t l0 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u), h0 = __builtin_amdgcn_perm(y[1], y[0], 0x07030602u);
  const uint32_t l1 = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u), h1 = __builtin_amdgcn_perm(y[3], y[2], 0x07030602u);
  d[0] = __builtin_amdgcn_perm(l1, l0, 0x05040100u) ^ 0x80808080u;
  d[1] = __builtin_amdgcn_perm(l1, l0, 0x07060302u) ^ 0x80808080u;
  d[2] = __builtin_amdgcn_perm(h1, h0, 0x05040100u) ^ 0x80808080u;
  d[3] = __builtin_amdgcn_perm(h1, h0, 0x07060302u) ^ 0x80808080u;
}
// Every plane of four words: d[p] holds their digits p.
template <typename T>
__device__ __forceinline__ void planes4(const T (&w)[4], uint32_t (&d)[sizeof(T)]) {
  uint32_t y[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = w[i] + 0x80808080u;
    bytes4(y, d);
  } else {
    uint32_t z[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint64_t v = w[i] + 0x8080808080808080ull;
      y[i] = uint32_t(v), z[i] = uint32_t(v >> 32);
    }
    bytes4(y, d);
    bytes4(z, d + 4);
  }
}
// 2^(8p) times a plane's sum
template <typename T>
__device__ __forceinline__ T plane_word(int32_t sum, int p) {
  return T(int64_t(sum)) << (8 * p);
}

// bytes of a row of weights that may be read: whole 16
__host__ __device__ __forceinline__ int q8_row(int K) { return (K + 15) & ~15; }

// Which of a column's 8 groups of 16 weights of a 128-k step lies where in LDS, for the
// reads' banks: column col of a tile of 16.
__device__ __forceinline__ int q8_turn(int col) {
  return (col >> 1 & 1) << 2 | (0x78 >> (col >> 2 << 1) & 3);
}

// ---------------------------------------------------------------------------
// Few rows, R at most: a workgroup takes 16 columns, its waves the 128-k steps of K in
// turn, each by itself: it asks for a step's weights, straight into its own part of LDS (in
// lines of memory; to the lanes' registers, 16 rows of them, they would take four times the
// cache's accesses), and words, one or, of few rows, two steps ahead (4096 x 11008: two of 8
// rows in Z_2^64 leave room for half as many waves, 30% slower; one of one row in Z_2^32 7%
// slower).  It forms the words' digits, four words a lane at a time, and turns them by its
// part of LDS into operands (formed in the lanes that need them, each word by as many
// lanes as there are planes or parts: 4096 x 11008, one row a third slower, 8 rows 60%).
// The waves' sums are added up through LDS.
// The MFMA's 16 rows are the words' by the planes' parts: of 8 words in Z_2^32, say, planes
// 0 and 1, then 2 and 3, so that a step has 2 R planes / 16 MFMAs.
// Places: a read of 16 bytes serves lanes 0-3, 12-15, 20-27 together, then 4-11, 16-19,
// 28-31; groups of 16 bytes are turned so that those fall into different banks.
// Bound by the weights' bytes and, below some 20 MB, by a launch's start and the waves'
// first loads: in Z_2^32 1 x 4096 x 4096 3.4 us with the weights in the card's cache and 5.3 with
// them in memory, 1 x 4096 x 11008 9.2 and 10.4, 1 x 8192 x 8192 13.0 and 14.2 (4.7 TB/s), 1 x 4096 x
// 32000 21.6 and 23.8 (5.5 TB/s); with more rows by the digits, which each workgroup forms, their way
// through LDS and the words' way to every CU: 4096 x 4096, 8 rows 5.3 and 7.0, 16 rows 7.5 and 8.8.
// ---------------------------------------------------------------------------
template <typename T, int R, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_q8_few(Q8Args<T> g) {
  constexpr int NP = int(sizeof(T)), MT = R > 16 ? R / 16 : 1;  // tiles of 16 rows
  constexpr int PARTS = MT > 1 ? 1 : 16 / R < NP ? 16 / R : NP, PW = NP / PARTS;  // planes of a part
  constexpr int NR = PARTS < 4 ? 4 / PARTS : 1;                // a lane's words of a tile of the output
  constexpr int QUADS = R / 2;                                 // a lane's groups of four words of a step
  constexpr int NW = 2, NB = QUADS * NP / 4;                   // loads of a step's weights and words
  constexpr int D = R <= 4 ? 2 : 1;                            // steps asked for ahead
  constexpr int DIGITS = R * NP * 128, OWN = D * NW * 1024 + DIGITS;  // bytes: of a step's digits, of a wave
  __shared__ __align__(16) uint8_t lds[WAVES * OWN];
  static_assert(sizeof lds >= WAVES * MT * NR * 64 * sizeof(T), "the sums' place");
  const int tid = int(threadIdx.x), lane = tid & 63, waves = int(blockDim.x) >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, lg = lane >> 4, n0 = int(blockIdx.x) * 16;
  uint8_t *own = lds + wave * OWN, *digits = own + D * NW * 1024;
  const int steps = (g.K + 127) / 128, whole = g.K / 128, end = q8_row(g.K) - 16, mine = (steps - wave + waves - 1) / waves;

  // what this lane asks for: 16 weights of columns lane / 8 and 8 + lane / 8, four words of
  // rows lane / 32 + 2 i
  const int nq = min(g.N - n0, 16), kq = lane % 32;
  const __amdgpu_buffer_rsrc_t qr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<int8_t *>(g.q + size_t(n0) * g.ldq), short(0), int(uint32_t(nq - 1) * uint32_t(g.ldq) + uint32_t(end + 16)),
      kRsrcWord3);
  const __amdgpu_buffer_rsrc_t ar = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<T *>(g.a), short(0), int((uint32_t(g.M - 1) * uint32_t(g.lda) + uint32_t(g.K)) * uint32_t(NP)), kRsrcWord3);
  uint32_t qo[NW], qk[NW], ao[QUADS], to[QUADS];
#pragma unroll
  for (int i = 0; i < NW; i++) {
    const int col = 8 * i + lane / 8;
    qo[i] = uint32_t(min(col, nq - 1)) * uint32_t(g.ldq);
    qk[i] = uint32_t(16 * ((lane % 8) ^ q8_turn(col)));
  }
#pragma unroll
  for (int i = 0; i < QUADS; i++) ao[i] = uint32_t(min(lane / 32 + 2 * i, g.M - 1)) * uint32_t(g.lda) * uint32_t(NP);
  // Digits: plane, row, 128 bytes; group j of 16 bytes at j ^ (the plane's part + PARTS (row / 2)) % 8.
#pragma unroll
  for (int i = 0; i < QUADS; i++) to[i] = uint32_t((lane / 32 + 2 * i) * 128 + kq % 4 * 4 + ((kq / 4) ^ (PARTS * i % 8)) * 16);
  const int row = R * PARTS < 16 ? li / PARTS % R : li / PARTS, part = li % PARTS;
  uint32_t fromw[2], from[2];
#pragma unroll
  for (int o = 0; o < 2; o++) {
    fromw[o] = uint32_t(li * 128 + ((4 * o + lg) ^ q8_turn(li)) * 16);
    from[o] = uint32_t((part * PW * R + row) * 128 + ((4 * o + lg) ^ (part + PARTS * (row / 2))) * 16);
  }

  struct Words {
    Four<T> w[QUADS];
  };
  auto ask = [&](int i, Words &x) __attribute__((always_inline)) {
    const int s = wave + i * waves;
#pragma unroll
    for (int j = 0; j < NW; j++)  // past the end of a row they meet words' zeros
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          qr, (__attribute__((address_space(3))) void *)(own + (i % D * NW + j) * 1024), 16,
          int(qo[j] + min(128 * s + qk[j], uint32_t(end))), 0, 0, 0);
    const uint32_t k = uint32_t(min(128 * s + 4 * kq, g.K - 4) * NP);  // past K: the last four, to be cut
#pragma unroll
    for (int j = 0; j < QUADS; j++)
#pragma unroll
      for (int h = 0; h < NP / 4; h++) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(ar, int(ao[j] + k + 16 * h), 0, 0);
        __builtin_memcpy(reinterpret_cast<uint8_t *>(x.w[j].w) + 16 * h, &v, 16);
      }
    __builtin_amdgcn_sched_barrier(0);  // here, not where they are used
  };

  v4i_t acc[MT][PW] = {};  // of at most 512 steps (launch_part), 2^16 terms
  // Step i of this wave, in x; `later` of its steps have been asked for since; more: x asks for step i + D.
  auto step = [&](int i, Words &x, auto later, auto more) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(later)::value * (NW + NB)) : "memory");
#pragma unroll
    for (int j = 0; j < QUADS; j++)  // not read before
#pragma unroll
      for (int k = 0; k < 4; k++) asm volatile("" : "+v"(x.w[j].w[k]));
    const int s = wave + i * waves;
    v4i_t b[2];
#pragma unroll
    for (int o = 0; o < 2; o++) b[o] = *reinterpret_cast<const v4i_t *>(own + (fromw[o] + uint32_t(i % D * NW * 1024)));
    if (s >= whole) {
#pragma unroll
      for (int j = 0; j < QUADS; j++) x.w[j].cut(128 * s + 4 * kq, g.K);
    }
#pragma unroll
    for (int j = 0; j < QUADS; j++) {
      uint32_t d[NP];
      planes4<T>(x.w[j].w, d);
#pragma unroll
      for (int p = 0; p < NP; p++)  // the part turns the groups: lanes' places differ by it in bits 4 to 6
        *reinterpret_cast<uint32_t *>(digits + ((to[j] ^ uint32_t(p / PW * 16)) + uint32_t(p * R * 128))) = d[p];
      __builtin_amdgcn_sched_barrier(0);  // left free, the compiler takes more registers than there are
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the weights have been read, the digits are there
    if constexpr (decltype(more)::value) ask(i + D, x);
#pragma unroll
    for (int o = 0; o < 2; o++)
#pragma unroll
      for (int k = 0; k < PW; k++)
#pragma unroll
        for (int t = 0; t < MT; t++)
          acc[t][k] = mfma64(*reinterpret_cast<const v4i_t *>(digits + (from[o] + uint32_t(k * R * 128 + t * 2048))), b[o],
                             acc[t][k]);
    __builtin_amdgcn_sched_barrier(0);  // before the next step's words are waited for
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  constexpr std::integral_constant<int, 0> none{};
  constexpr std::integral_constant<int, 1> one{};
  // this thread's word of the output, and its scales
  const int n = n0 + tid % 16;
  const int32_t sn = g.scale ? g.scale[min(n, g.N - 1)] : 1;
  int32_t sm = g.tok ? g.tok[min(tid / 16, g.M - 1)] : 1;
  if constexpr (D == 1) {
    Words x;
    ask(0, x);
    for (int i = 0; i + 1 < mine; i++) step(i, x, none, yes);
    step(mine - 1, x, none, no);
  } else {  // no branch of fewer loads before a load's use: behind it the compiler would wait for all
    Words x, y;
    ask(0, x);
    if (mine > 1) {
      ask(1, y);
      int i = 0;
      for (; i + 3 < mine; i += 2) {
        step(i, x, one, yes);
        step(i + 1, y, one, yes);
      }
      if (i + 2 < mine) {
        step(i, x, one, yes);
        step(i + 1, y, one, no);
        y = x;
      } else {
        step(i, x, one, no);
      }
    } else {
      y = x;
    }
    step(mine - 1, y, none, no);
  }
  // a register's row of 4: part j % PARTS of a word; of eight parts, the upper four where lg is odd
  T out[MT * NR] = {};
#pragma unroll
  for (int t = 0; t < MT; t++)
#pragma unroll
    for (int k = 0; k < PW; k++)
#pragma unroll
      for (int j = 0; j < 4; j++) out[t * NR + j / (4 / NR)] += plane_word<T>(acc[t][k][j], j % (4 / NR) * PW + k);
  __syncthreads();
  T *red = reinterpret_cast<T *>(lds);  // wave, register, lane
#pragma unroll
  for (int r = 0; r < MT * NR; r++) red[(wave * MT * NR + r) * 64 + lane] = out[r];
  __syncthreads();
  for (int r = tid / 16; r < min(R, g.M); r += 4 * waves) {
    T v = 0;
    for (int w = 0; w < waves; w++) {
      const T *z = red + w * MT * NR * 64 + tid % 16;
      if constexpr (PARTS <= 4) v += z[(r / 16 * NR + r % NR) * 64 + 16 * (r % 16 / NR)];
      else v += z[32 * r] + (z[32 * r + 16] << 32);
    }
    if (n < g.N) g.c[size_t(r) * g.ldc + n] = v * T(int64_t(sn)) * T(int64_t(sm));
    if (g.tok) sm = g.tok[min(r + 4 * waves, g.M - 1)];
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of 2 x 4 waves takes a tile of TILES times 16 words by 64 NT columns,
// 128 k a step: 64 or 32 words of Z_2^32, 32 or 16 of Z_2^64, whose planes the two rows of waves
// share where there are but 16.
// It forms the words' digits once, for the next step between the matrix instructions of
// this one; the weights go straight into LDS (to the lanes' registers they would take four
// times the cache's accesses: an operand's 16 rows are as many places for 16 lanes, where here
// 8 lanes take a row's 128 bytes: 29% slower).  1000 x 4096 x 4096 in Z_2^32: 61 to 72 us by
// the card, 1.9 to 2.2 POP/s of digits (a large int8 library product 2.0 to 2.1).  32 steps take
// 1.7 us each, the start and the output's way to memory 8.  The matrix cores are busy half of
// that (the same instructions from registers take 34 to 41 us); the rest is one workgroup of two waves a
// SIMD that waits at a barrier each step for loads, digits and reads of LDS.  Words or weights of
// zeros take 54 us where uniform ones take 62: of the rest the card's power is the smaller part.
// Places in LDS, both such that neither the writes' nor the reads' lanes meet in a bank
// (a read of 16 bytes serves lanes 0-3, 12-15, 20-27 together, then 4-11, 16-19, 28-31):
//   digits   plane, tile of 16 words, half of the step o: 64 lanes' 16 bytes, word li of
//            lane group lg at li ^ 2 (4 o + lg);
//   weights  8 columns: a column's 8 groups of 16 k, group o 4 + lg at that ^ q8_turn.
// K may be split over workgroups, which then add to a cleared output: sums modulo 2^bw do
// not depend on their order.
// ---------------------------------------------------------------------------
template <typename T, int TILES, int NT>
__global__ __launch_bounds__(512, NT >= 2 ? 2 : 4) void k_q8_many(Q8Args<T> g, int rows, int cols, int splits) {
  constexpr int NP = int(sizeof(T)), BM = 16 * TILES, QUADS = BM * 32 / 512;
  constexpr bool SHARED = TILES == 1;                              // a wave has half of the planes
  constexpr int MT = SHARED ? 1 : TILES / 2, PW = SHARED ? NP / 2 : NP;  // a wave's tiles and planes
  constexpr int PLANE = TILES * 2 * 1024, WORDS = NP * PLANE, WEIGHTS = 64 * NT * 128;  // bytes
  constexpr int WB = 3;  // steps of weights in LDS: in use, there, on their way
  __shared__ __align__(16) uint8_t lds[2 * WORDS + WB * WEIGHTS];
  const int at = xcd_swizzle(int(blockIdx.x), int(gridDim.x));
  // tiles in bands of 8 rows, column by column: an XCD's consecutive tiles share rows and
  // columns (1000 x 4096 x 4096 1.6 us less than down all rows)
  const int split = at % splits, tile = at / splits, band = tile / (8 * cols), in = tile % (8 * cols);
  const int high = min(8, rows - 8 * band), m0 = (8 * band + in % high) * BM, n0 = in / high * 64 * NT;
  const int tid = int(threadIdx.x), lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 2, wn = wave & 3;
  const int wrow = SHARED ? 0 : wm * MT;  // the wave's first tile
  const int all = (g.K + 127) / 128, s0 = int(int64_t(all) * split / splits), s1 = int(int64_t(all) * (split + 1) / splits);
  const int end = q8_row(g.K) - 16;
  // This thread's groups of four words: rows tid / 32 + 16 i, k 4 (tid % 32).  A row's place is
  // 32 bits from one that the workgroup shares (launch_gemm_q8 bounds the strides).
  const int kq = tid % 32, j = kq / 4;  // j: 4 o + lg of the group
  const T *a[QUADS];
  uint32_t ao[QUADS];
#pragma unroll
  for (int i = 0; i < QUADS; i++) {
    const int r = min(m0 + 16 * i, g.M - 1);
    a[i] = g.a + size_t(r) * g.lda;
    ao[i] = uint32_t(min(tid / 32, g.M - 1 - r)) * uint32_t(g.lda) + uint32_t(4 * kq);
  }
  const uint32_t to = uint32_t((j * 16 + ((tid / 32) ^ (2 * j))) * 16 + kq % 4 * 4);
  // this lane's group of 16 weights of 8 columns, of NT such: column lane / 8 of the wave's
  // 8 columns i
  const int8_t *q = g.q + size_t(n0) * g.ldq;
  const int nq = min(g.N - n0, 64 * NT);
  const __amdgpu_buffer_rsrc_t qr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<int8_t *>(q), short(0), int(uint32_t(nq - 1) * uint32_t(g.ldq) + uint32_t(end + 16)), kRsrcWord3);
  uint32_t qo[NT], qk[NT];
#pragma unroll
  for (int i = 0; i < NT; i++) {
    const int col = (wave * NT + i) * 8 + lane / 8;
    qk[i] = uint32_t(16 * ((lane % 8) ^ q8_turn(col % 16)));
    qo[i] = uint32_t(min(col, nq - 1)) * uint32_t(g.ldq);
  }
  uint32_t from[2], fromw[2];
#pragma unroll
  for (int o = 0; o < 2; o++) {
    from[o] = uint32_t((o * 64 + lg * 16 + (li ^ (2 * (4 * o + lg)))) * 16 + wm * (SHARED ? PW * PLANE : MT * 2048));
    fromw[o] = uint32_t(2 * WORDS + wn * NT * 2048 + li * 128 + ((4 * o + lg) ^ q8_turn(li)) * 16);
  }

  v4i_t acc[MT][PW][NT] = {};
  struct Words {
    Four<T> w[QUADS];
  };
  const int whole = min(s1, g.K / 128);  // steps up to here are within K
  auto load_words = [&](int s, Words &x, int i) __attribute__((always_inline)) {  // of a step within K
    __builtin_memcpy(x.w[i].w, a[i] + 128 * s + ao[i], sizeof x.w[i].w);
  };
  auto load_last = [&](int s, Words &x) __attribute__((always_inline)) {  // to be cut
#pragma unroll
    for (int i = 0; i < QUADS; i++) x.w[i].load(a[i] + (ao[i] - 4 * kq), 128 * s + 4 * kq, g.K);
  };
  auto cut = [&](int s, Words &x) __attribute__((always_inline)) {
    if (s < whole) return;
#pragma unroll
    for (int i = 0; i < QUADS; i++) x.w[i].cut(128 * s + 4 * kq, g.K);
  };
  auto load_weights = [&](int s, int buf, auto within) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
      auto *to = (__attribute__((address_space(3))) void *)(lds + 2 * WORDS + buf * WEIGHTS + (wave * NT + i) * 1024);
      if constexpr (decltype(within)::value)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(qr, to, 16, int(qo[i] + qk[i]), 128 * s, 0, 0);
      else  // past the end of a row they meet words' zeros
        __builtin_amdgcn_raw_ptr_buffer_load_lds(qr, to, 16, int(qo[i] + min(128 * s + qk[i], uint32_t(end))), 0, 0, 0);
    }
  };
  auto put = [&](int buf, const Words &x, int i) __attribute__((always_inline)) {
    uint32_t d[NP];
    planes4<T>(x.w[i].w, d);
#pragma unroll
    for (int p = 0; p < NP; p++) *reinterpret_cast<uint32_t *>(lds + to + (buf * WORDS + p * PLANE + i * 2048)) = d[p];
  };
  // This wave's LDS accesses are done, its loads into LDS (which the compiler does not wait
  // for) but for the last `later` loads among them, and every wave's.
  auto barrier = [&](auto later) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(later)::value) : "memory");
  };
  constexpr std::integral_constant<int, 0> none{};
  // The products of a step, an operand of words read ahead; between them, a few
  // instructions for each operand, the next step's words become digits (more).  The order
  // is held: left free, the compiler reads so far ahead that registers spill.
  constexpr int F = 2 * PW * MT;           // operands of words
  constexpr int STAGES = F / QUADS;        // operands by the time of a group of four words
  static_assert(STAGES == NP, "four planes take four stages");
  struct Turning {
    uint32_t y[4], z[4], l[2], h[2];
  };
  auto turn = [&](int buf, const Words &x, Turning &v, int i, int stage) __attribute__((always_inline)) {
    uint8_t *p = lds + to + (buf * WORDS + i * 2048 + (stage & 4) * PLANE);
    if (stage == 0) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (NP == 4) {
          v.y[k] = x.w[i].w[k] + 0x80808080u;
        } else {
          const uint64_t u = x.w[i].w[k] + 0x8080808080808080ull;
          v.y[k] = uint32_t(u), v.z[k] = uint32_t(u >> 32);
        }
      }
    } else if (stage % 4 == 1) {
      const uint32_t(&y)[4] = stage & 4 ? v.z : v.y;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        v.l[k] = __builtin_amdgcn_perm(y[2 * k + 1], y[2 * k], 0x05010400u);
        v.h[k] = __builtin_amdgcn_perm(y[2 * k + 1], y[2 * k], 0x07030602u);
      }
    } else if (stage != 4) {
      const uint32_t(&u)[2] = stage & 1 ? v.h : v.l;
      p += (stage & 1) * 2 * PLANE;
      *reinterpret_cast<uint32_t *>(p) = __builtin_amdgcn_perm(u[1], u[0], 0x05040100u) ^ 0x80808080u;
      *reinterpret_cast<uint32_t *>(p + PLANE) = __builtin_amdgcn_perm(u[1], u[0], 0x07060302u) ^ 0x80808080u;
    }
  };
  auto compute = [&](int buf, int wbuf, const Words &x, auto more) __attribute__((always_inline)) {
    v4i_t b[NT];
    Turning v;
    auto operand = [&](int f) __attribute__((always_inline)) {
      return *reinterpret_cast<const v4i_t *>(lds + from[f / (PW * MT)] +
                                              (buf * WORDS + f / MT % PW * PLANE + f % MT * 2048));
    };
    v4i_t d = operand(0);
#pragma unroll
    for (int f = 0; f < F; f++) {
      const int o = f / (PW * MT), p = f / MT % PW, i = f % MT;
      if (f % (PW * MT) == 0) {
#pragma unroll
        for (int t = 0; t < NT; t++)
          b[t] = *reinterpret_cast<const v4i_t *>(lds + (fromw[o] + uint32_t(wbuf * WEIGHTS)) + t * 2048);
      }
      v4i_t ahead = d;
      if (f + 1 < F) ahead = operand(f + 1);
      if constexpr (decltype(more)::value) turn(buf ^ 1, x, v, f / STAGES, f % STAGES);
#pragma unroll
      for (int t = 0; t < NT; t++) acc[i][p][t] = mfma64(d, b[t], acc[i][p][t]);
      d = ahead;
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  // Words and weights are asked for two steps ahead: words have a step to come and are then
  // turned, weights have two.  Steps within K have no branch between a load and its use (at a
  // join the compiler waits for all of them); a last step past K has its words cut.
  Words x, y;
  auto any_words = [&](int s, Words &v) __attribute__((always_inline)) {
    if (s < whole) {
#pragma unroll
      for (int i = 0; i < QUADS; i++) load_words(s, v, i);
    } else if (s < s1) {
      load_last(s, v);
    }
  };
  auto put_all = [&](int buf, const Words &v) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QUADS; i++) put(buf, v, i);
  };
  load_weights(s0, 0, no);
  if (s0 + 1 < s1) load_weights(s0 + 1, 1, no);
  int32_t sn[NT], sm[MT][4];
#pragma unroll
  for (int t = 0; t < NT; t++) sn[t] = g.scale ? g.scale[min(n0 + (wn * NT + t) * 16 + li, g.N - 1)] : 1;
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) sm[i][r] = g.tok ? g.tok[min(m0 + (wrow + i) * 16 + 4 * lg + r, g.M - 1)] : 1;
  {
    Words first;
    any_words(s0, first);
    any_words(s0 + 1, x);
    cut(s0, first);
    put_all(0, first);
  }
#pragma unroll
  for (int t = 0; t < NT; t++) asm volatile("" : "+v"(sn[t]));  // here, not where they are used
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) asm volatile("" : "+v"(sm[i][r]));
  barrier(none);
  int s = s0, wb = 0, wnext = 2;  // buffers of this step's weights and of those asked for next
  auto turn_buffers = [&]() {
    s++;
    wb = wb == WB - 1 ? 0 : wb + 1;
    wnext = wnext == WB - 1 ? 0 : wnext + 1;
  };
  auto step = [&](auto buf, Words &cur, Words &ahead) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QUADS; i++)  // here, so that their use does not wait for the loads that leave next
#pragma unroll
      for (int k = 0; k < 4; k++) asm volatile("" : "+v"(cur.w[i].w[k]));
#pragma unroll
    for (int i = 0; i < QUADS; i++) load_words(s + 2, ahead, i);
    load_weights(s + 2, wnext, yes);
    __builtin_amdgcn_sched_barrier(0);  // asked for here, not where they are used
    compute(buf, wb, cur, yes);
    // the next step's weights are older than these loads, at least one for each 16 bytes
    barrier(std::integral_constant<int, QUADS * int(sizeof(T)) / 4 + NT>{});
    turn_buffers();
  };
  while (s + 3 < whole) {
    step(std::integral_constant<int, 0>{}, x, y);
    step(std::integral_constant<int, 1>{}, y, x);
  }
  // the last three or fewer
  for (int buf = 0; s < s1; turn_buffers(), buf ^= 1) {
    if (s + 2 < s1) load_weights(s + 2, wnext, no);
    compute(buf, wb, x, no);
    if (s + 1 < s1) {
      cut(s + 1, x);
      put_all(buf ^ 1, x);
      any_words(s + 2, x);
      barrier(none);
    }
  }

  uint32_t *upper = reinterpret_cast<uint32_t *>(lds);  // shared planes: a word's upper half
  if constexpr (SHARED) {
    barrier(none);  // the last step's operands have been read
    if (wm == 1) {
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          uint32_t v = 0;
#pragma unroll
          for (int p = 0; p < PW; p++) v += uint32_t(acc[0][p][t][r]) << (8 * p);
          upper[((wn * NT + t) * 4 + r) * 64 + lane] = v;
        }
    }
    barrier(none);
    if (wm == 1) return;
  }
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int m = m0 + (wrow + i) * 16 + 4 * lg + r;
      if (m >= g.M) continue;
      T *c = g.c + size_t(m) * g.ldc;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const int n = n0 + (wn * NT + t) * 16 + li;
        T v = 0;
#pragma unroll
        for (int p = 0; p < PW; p++) v += plane_word<T>(acc[i][p][t][r], p);
        if constexpr (SHARED) v += T(upper[((wn * NT + t) * 4 + r) * 64 + lane]) << 32;
        v *= T(int64_t(sn[t])) * T(int64_t(sm[i][r]));
        if (n >= g.N) continue;
        if (splits == 1) {
          c[n] = v;
        } else {
          using W = std::conditional_t<sizeof(T) == 4, unsigned, unsigned long long>;
          atomicAdd(reinterpret_cast<W *>(c + n), W(v));
        }
      }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_q8_clear(Q8Args<T> g) {
  const size_t n = size_t(g.M) * size_t(g.N);
  for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += size_t(gridDim.x) * 256)
    g.c[i / g.N * g.ldc + i % g.N] = 0;
}

// The weights' way from memory (us), at 6.5 TB/s (in part from the card's cache).
template <typename T>
float weights_time(const Q8Args<T> &g) {
  return float(g.K) * float(g.N) / 6.5e6f;
}
// What a launch of k_q8_few takes (us): its start and the larger of the weights' way and its
// rounds of one workgroup a CU times a wave's steps, each the digits of R rows and, with more
// than half of the CUs at work, the words' way to them; where but one workgroup fits a CU each
// round has a start.  Fitted to weights in the card's cache, as the rule's other side is.  Both kernels,
// few and many rows' (us, weights in the cache; then in memory):
//   Z_2^32   1 row     4096 x 4096 3.4 and 7.6; 5.3, 8.8      4096 x 32000 22.4 and 23.9; 24.7, 28.3
//            4 rows    4096 x 4096 4.1 and 8.9; 5.7, 10.0     4096 x 32000 23.0 and 25.3; 26.0, 29.8
//            8 rows    4096 x 4096 5.3 and 9.2; 7.0, 10.0     8192 x 8192 14.5 and 17.3; 18.7, 18.8
//                      20000 x 300 11.0 and 8.3; 20.7, 9.5    20000 x 4096 16.4 and 20.0; 24.6, 22.8
//            16 rows   4096 x 4096 7.5 and 9.8; 8.9, 10.4     8192 x 300 8.8 and 7.2; 12.8, 8.0
//                      8192 x 2500 10.6 and 12.3; 13.4, 12.8
//            32 rows   1024 x 1024 4.4 and 6.8; 5.3, 7.6      2048 x 4096 7.3 and 7.7; 7.9, 8.5
//                      4096 x 4096 12.1 and 10.8; 13.5, 11.7  1000 x 4099 8.5 and 7.5; 9.7, 8.8
//   Z_2^64   1 row     4096 x 4096 4.3 and 7.9; 6.0, 9.1
//            4 rows    8192 x 8192 14.2 and 18.2; 18.3, 20.2  20000 x 300 10.6 and 8.0; 21.5, 9.3
//            8 rows    4096 x 4096 7.6 and 9.8; 9.0, 10.4     8192 x 2500 10.6 and 11.3; 13.4, 12.1
//            16 rows   1024 x 1024 4.4 and 6.9; 5.4, 7.8      2048 x 2048 6.2 and 7.2; 7.6, 8.1
//                      4096 x 4096 12.2 and 10.9; 13.6, 12.0
// With them in memory a long K of 6 to 16 rows is up to 11% faster by the other kernel.
template <typename T>
float few_time(const Launch &L, const Q8Args<T> &g) {
  const float digits = float(sizeof(T)) * (g.M <= 2 ? 2.f : g.M <= 4 ? 4.f : g.M <= 8 ? 8.f : g.M <= 16 ? 16.f : 32.f);
  const float wgs = std::ceil(float(g.N) / 16), cus = float(L.num_cu), rounds = std::ceil(wgs / cus);
  const float step = 0.15f + 0.0125f * digits + 0.006f * digits * std::max(0.f, 2 * std::min(1.f, wgs / cus) - 1);
  return 2.5f + std::max(rounds * std::ceil(float(g.K) / 1024) * step, weights_time(g)) +
         (digits >= 128 ? 2.2f * (rounds - 1) : 0.f);
}
template <typename T>
hipError_t launch_few(const Launch &L, const Q8Args<T> &g) {
  const int steps = (g.K + 127) / 128;
  auto few = [&](auto rows, auto most) {
    constexpr int WAVES = decltype(most)::value;
    hipLaunchKernelGGL((k_q8_few<T, decltype(rows)::value, WAVES>), dim3(unsigned((g.N + 15) / 16)),
                       dim3(64u * unsigned(std::min(steps, WAVES))), 0, L.stream, g);
    return hipGetLastError();
  };
  constexpr std::integral_constant<int, 2> two{};
  constexpr std::integral_constant<int, 4> four{};
  constexpr std::integral_constant<int, 8> eight{};
  constexpr std::integral_constant<int, 16> sixteen{};
  if constexpr (sizeof(T) == 4) {
    if (g.M > 16) return few(std::integral_constant<int, 32>{}, eight);
  }
  if (g.M > 4) return g.M <= 8 ? few(eight, eight) : few(sixteen, eight);
  // Sixteen waves where they have a step each and a workgroup has a CU (us, Z_2^32, by eight
  // and by sixteen; with the weights in memory): one row of 4096 x 4096 3.6 and 3.4; 5.7, 5.3, of 8192 x
  // 2048 4.5 and 4.3; 6.2, 6.2; four of 4096 x 4096 4.1 and 4.2; 6.1, 5.7, of 8192 x 4096 8.2 and 7.4; 9.0,
  // 8.4, of 4096 x 11008 9.3 and 11.3; 11.4, 13.3, of 1000 x 4099 2.7 and 3.5; 3.7, 4.6.
  if (steps > 8 && g.N <= 16 * L.num_cu) return g.M <= 2 ? few(two, sixteen) : few(four, sixteen);
  return g.M <= 2 ? few(two, eight) : few(four, eight);
}

template <typename T>
constexpr int kLarge = 16 / int(sizeof(T));  // tiles of 16 words of a large tile of k_q8_many
template <typename T>
hipError_t launch_part(const Launch &L, const Q8Args<T> &g) {
  constexpr int NP = int(sizeof(T));
  const int steps = (g.K + 127) / 128, exact = (steps + kExact / 128 - 1) / (kExact / 128);
  // The tile and the parts of K for which a launch takes least: its rounds of one workgroup a
  // CU, each with its start and its steps (two workgroups of the smallest tiles fit a CU, and
  // start together), and, where K is split, the output's clearing and the sums' way through
  // memory.  Measured (us, one MI355X, all CUs at work): a large tile's step 0.6 + 0.3 nt, its
  // start 6; a small one's 0.27 + 0.19 nt and 4; splitting 2.5, 0.1 a part and 0.25 a MB.  4096 x 4096 in
  // Z_2^32 by small tiles of width 1, 2, 3, 4 and by large ones of 3, 4: 1000 rows 115, 81, 87, 75 and
  // 91, 63; 640 75, 58, 59, 66 and 48, 55; 512 59, 42, 57, 38 and 45, 54; 256 31, 25, 29, 33 and 44, 53; 64
  // rows by four parts of K 13, 13, 14, 14 and 19, 21.
  int nt = 1, splits = exact;
  bool large = false;
  float best = 0;
  for (int big = 0; big < 2; big++)
    for (int w = big ? 3 : 1; w <= 4; w++)  // narrower large tiles take longer than wider small ones
      for (int p = exact; p == exact || (p <= steps / 4 && p <= 64); p *= 2) {
        const int words = big ? kLarge<T> * 16 : kLarge<T> * 8;
        const float tiles = float((g.M + words - 1) / words) * float((g.N + 64 * w - 1) / (64 * w)) * float(p);
        const float rounds = std::ceil(tiles / float(L.num_cu)), starts = !big && w <= 2 ? 1.f : rounds;
        const float step = big ? 0.6f + 0.3f * float(w) : 0.27f + 0.19f * float(w);
        float t = starts * (big ? 6.f : 4.f) + rounds * float((steps + p - 1) / p) * step;
        if (p > 1) t += 2.5f + 0.1f * float(p) + 0.25e-6f * float(g.M) * float(g.N) * float(p * NP);
        if (best == 0 || t < best) best = t, nt = w, splits = p, large = big != 0;
      }
  // few rows: four words to load, plane sums in 32 bits
  if (g.M <= 128 / NP && g.K >= 4 && steps <= 8 * (kExact / 128) && few_time(L, g) <= std::max(best, 4 + weights_time(g)))
    return launch_few<T>(L, g);
  const int words = large ? kLarge<T> * 16 : kLarge<T> * 8, rows = (g.M + words - 1) / words;
  const int cols = (g.N + 64 * nt - 1) / (64 * nt);
  const size_t wgs = size_t(rows) * size_t(cols) * size_t(splits);
  if (wgs > kMostThreads / 512) return hipErrorInvalidValue;  // more memory than there is
  if (splits > 1) {
    const size_t want = (size_t(g.M) * size_t(g.N) + 255) / 256;
    hipLaunchKernelGGL((k_q8_clear<T>), dim3(unsigned(std::min(want, size_t(L.num_cu) * 8))), dim3(256), 0, L.stream, g);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  auto many = [&](auto tiles, auto w) {
    hipLaunchKernelGGL((k_q8_many<T, decltype(tiles)::value, decltype(w)::value>), dim3(unsigned(wgs)), dim3(512), 0, L.stream, g,
                       rows, cols, splits);
    return hipGetLastError();
  };
  constexpr std::integral_constant<int, kLarge<T>> most{};
  constexpr std::integral_constant<int, kLarge<T> / 2> half{};
  switch (nt) {
    case 1: return many(half, std::integral_constant<int, 1>{});
    case 2: return many(half, std::integral_constant<int, 2>{});
    case 3: return large ? many(most, std::integral_constant<int, 3>{}) : many(half, std::integral_constant<int, 3>{});
    default: return large ? many(most, std::integral_constant<int, 4>{}) : many(half, std::integral_constant<int, 4>{});
  }
}

// rows m.. and columns n.. of a product
template <typename T>
Q8Args<T> part(const Q8Args<T> &g, int64_t m, int rows, int64_t n, int cols) {
  Q8Args<T> p = g;
  p.M = int(std::min<int64_t>(g.M - m, rows));
  p.N = int(std::min<int64_t>(g.N - n, cols));
  p.a += size_t(m) * g.lda;
  p.q += size_t(n) * g.ldq;
  if (p.scale) p.scale += n;
  if (p.tok) p.tok += m;
  p.c += size_t(m) * g.ldc + size_t(n);
  return p;
}

}  // namespace

template <typename T>
hipError_t launch_gemm_q8(const Launch &L, const Q8Args<T> &g) {
  if (g.K > kQ8MaxK) return hipErrorInvalidValue;
  // Rows' places are 32 bits from what a workgroup shares: rows that lie further apart are
  // taken one by one, weights in columns of their own.
  const bool far_a = g.lda >= size_t(1) << 24, far_q = g.ldq >= size_t(1) << 23;
  if ((far_a && g.M > 1) || (far_q && g.N > 1)) {
    const int rows = far_a ? 1 : g.M, cols = far_q ? 1 : g.N;
    for (int64_t m = 0; m < g.M; m += rows)
      for (int64_t n = 0; n < g.N; n += cols) {
        Q8Args<T> p = part(g, m, rows, n, cols);
        p.lda = p.M == 1 ? size_t(p.K) : p.lda;
        p.ldq = p.N == 1 ? size_t(q8_row(p.K)) : p.ldq;
        const hipError_t e = launch_gemm_q8<T>(L, p);
        if (e != hipSuccess) return e;
      }
    return hipSuccess;
  }
  // HIP cuts a launch of 2^32 threads along a dimension short: in parts of at most 2^13
  // rows by 2^18 columns, 2^9 by 2^12 tiles of 512 threads, of fewer columns where K is
  // split in 2^16s, the grid stays below that.
  const int rows = 1 << 13, cols = std::max(64, (1 << 18) / ((g.K + kExact - 1) / kExact));
  for (int64_t m = 0; m < g.M; m += rows)
    for (int64_t n = 0; n < g.N; n += cols) {
      const hipError_t e = launch_part<T>(L, part(g, m, rows, n, cols));
      if (e != hipSuccess) return e;
    }
  return hipSuccess;
}
template hipError_t launch_gemm_q8<uint32_t>(const Launch &, const Q8Args<uint32_t> &);
template hipError_t launch_gemm_q8<uint64_t>(const Launch &, const Q8Args<uint64_t> &);

}  // namespace mpcx
