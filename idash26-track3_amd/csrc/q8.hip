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
#include <type_traits>

#include "attn.h"
#include "digits.h"
#include "launch_util.h"

namespace mpcx {
namespace {

constexpr int kExact = 1 << 16;  // terms of a 32-bit plane sum

__device__ __forceinline__ v4i_t mfma64(v4i_t a, v4i_t b, v4i_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// Four words of a row from k on, zero from K on; rows start at any word, so the loads of
// 16 bytes are not assumed aligned to more than a word.
template <typename T>
__device__ __forceinline__ void load4(const T *row, int k, int K, T (&w)[4]) {
  if (k + 4 <= K) {
    __builtin_memcpy(w, row + k, sizeof w);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = k + i < K ? row[k + i] : T(0);
  }
}
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
// Plane p (a lane's own) of four words.
template <typename T>
__device__ __forceinline__ uint32_t plane4(const T (&w)[4], int p) {
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      y[i] = w[i] + 0x80808080u;
    } else {
      const uint64_t v = w[i] + 0x8080808080808080ull;
      y[i] = p & 4 ? uint32_t(v >> 32) : uint32_t(v);
    }
  }
  const uint32_t b = uint32_t(p & 3), sel = b | (b + 4) << 8;
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], sel), __builtin_amdgcn_perm(y[1], y[0], sel),
                               0x05040100u) ^
         0x80808080u;
}
// 2^(8p) times a plane's sum
template <typename T>
__device__ __forceinline__ T plane_word(int32_t sum, int p) {
  return T(int64_t(sum)) << (8 * p);
}

// bytes of a row of weights that may be read: whole 16
__device__ __forceinline__ int q8_row(int K) { return (K + 15) & ~15; }

template <typename T>
__device__ __forceinline__ T scaled(const Q8Args<T> &g, T v, int m, int n) {
  if (g.scale) v *= T(int64_t(g.scale[n]));
  if (g.tok) v *= T(int64_t(g.tok[m]));
  return v;
}

// ---------------------------------------------------------------------------
// Few rows: a workgroup takes 16 columns, its (up to 16) waves the 128-k steps of K in turn
// and add up their sums through LDS; each lane forms its digits from the words.  PACKED
// (rows <= 16 / planes): the MFMA's 16 rows are all planes of those words.  Else its rows
// are the words and each plane has an MFMA of its own, whose operands a lane forms together.
// ---------------------------------------------------------------------------
template <typename T, bool PACKED>
__global__ __launch_bounds__(1024) void k_q8_few(Q8Args<T> g) {
  constexpr int NP = int(sizeof(T)), NA = PACKED ? 1 : NP;
  __shared__ T red[16][PACKED ? 1 : 4][64];
  const int tid = int(threadIdx.x), lane = tid & 63, waves = int(blockDim.x) >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, lg = lane >> 4;
  const int n = int(blockIdx.x) * 16 + li;
  const int8_t *q = g.q + size_t(min(n, g.N - 1)) * g.ldq;
  const int m = PACKED ? li / NP : li;
  const T *a = g.a + size_t(min(m, g.M - 1)) * g.lda;
  const int steps = (g.K + 127) / 128, end = q8_row(g.K) - 16;
  T out[PACKED ? 1 : 4] = {};
  for (int s0 = wave; s0 < steps; s0 += kExact / 128 * waves) {
    v4i_t acc[NA] = {};
    const int s1 = min(steps, s0 + kExact / 128 * waves);
#pragma unroll 2
    for (int s = s0; s < s1; s += waves) {
      v4i_t b[2];
#pragma unroll
      for (int o = 0; o < 2; o++)  // past the end of a row they meet words' zeros
        b[o] = *reinterpret_cast<const v4i_t *>(q + min(128 * s + 64 * o + 16 * lg, end));
#pragma unroll
      for (int o = 0; o < 2; o++) {
        v4i_t d[NA];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          T w[4];
          load4<T>(a, 128 * s + 64 * o + 16 * lg + 4 * i, g.K, w);
          if constexpr (PACKED) {
            d[0][i] = int(plane4<T>(w, li % NP));
          } else {
            uint32_t p[NP];
            planes4<T>(w, p);
#pragma unroll
            for (int j = 0; j < NP; j++) d[j][i] = int(p[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < NA; j++) acc[j] = mfma64(d[j], b[o], acc[j]);
      }
    }
    if constexpr (PACKED) {  // four planes of one word; Z_2^64: the upper four where lg is odd
#pragma unroll
      for (int r = 0; r < 4; r++) out[0] += plane_word<T>(acc[0][r], r);
    } else {
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int j = 0; j < NP; j++) out[r] += plane_word<T>(acc[j][r], j);
    }
  }
#pragma unroll
  for (int r = 0; r < (PACKED ? 1 : 4); r++) red[wave][r][lane] = out[r];
  __syncthreads();
  constexpr int R = PACKED ? 16 / NP : 16;  // words of the tile
  for (int e = tid; e < R * 16; e += int(blockDim.x)) {
    const int r = e / 16, col = e % 16, on = int(blockIdx.x) * 16 + col;
    T v = 0;
    for (int w = 0; w < waves; w++) {
      if constexpr (!PACKED) v += red[w][r % 4][16 * (r / 4) + col];
      else if constexpr (NP == 4) v += red[w][0][16 * r + col];
      else v += red[w][0][32 * r + col] + (red[w][0][32 * r + 16 + col] << 32);
    }
    if (r < g.M && on < g.N) g.c[size_t(r) * g.ldc + on] = scaled<T>(g, v, r, on);
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of 2 x 4 waves takes 32 MT words by 64 NT columns.  A step is 128
// k, double-buffered in LDS and asked for a step ahead.  The workgroup forms the words'
// digits once; the weights go straight into LDS (to the lanes' registers they would take
// four times as long: the 16 rows of an operand are as many places in memory for each
// group of 16 lanes, where here 8 lanes take a row's 128 bytes).
// Places in LDS, both such that neither the writes' nor the reads' lanes meet in a bank
// (a read of 16 bytes serves lanes 0-3, 12-15, 20-27 together, then 4-11, 16-19, 28-31):
//   digits   plane, tile of 16 words, half of the step o: 64 lanes' 16 bytes, word li of
//            lane group lg at li ^ 2 (4 o + lg);
//   weights  8 columns: a column's 8 groups of 16 k, group o 4 + lg at that ^ q8_turn.
// K may be split over workgroups, which then add to a cleared output: sums modulo 2^bw do
// not depend on their order.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int q8_turn(int col) {  // of column col of a tile of 16
  return (col >> 1 & 1) << 2 | (0x78 >> (col >> 2 << 1) & 3);
}
template <typename T, int MT, int NT>
__global__ __launch_bounds__(512, NT >= 2 ? 2 : 4) void k_q8_many(Q8Args<T> g, int rows, int cols, int splits) {
  constexpr int NP = int(sizeof(T)), TILES = 2 * MT, BM = 16 * TILES, QUADS = BM * 32 / 512;
  constexpr int PLANE = TILES * 2 * 1024, WORDS = NP * PLANE, WEIGHTS = 64 * NT * 128;  // bytes
  __shared__ __align__(16) uint8_t lds[2][WORDS + WEIGHTS];
  const int at = xcd_swizzle(int(blockIdx.x), int(gridDim.x));
  const int split = at % splits, m0 = at / splits % rows * BM, n0 = at / splits / rows * 64 * NT;
  const int tid = int(threadIdx.x), lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 2, wn = wave & 3;
  const int all = (g.K + 127) / 128, s0 = int(int64_t(all) * split / splits), s1 = int(int64_t(all) * (split + 1) / splits);
  const int end = q8_row(g.K) - 16;
  // this thread's groups of four words: rows tid / 32 + 16 i, k 4 (tid % 32)
  const int kq = tid % 32, j = kq / 4;  // j: 4 o + lg of the group
  const T *a[QUADS];
  uint32_t to[QUADS];
#pragma unroll
  for (int i = 0; i < QUADS; i++) {
    const int r = tid / 32 + 16 * i;
    a[i] = g.a + size_t(min(m0 + r, g.M - 1)) * g.lda;
    to[i] = uint32_t(((r / 16 * 2 + j / 4) * 64 + j % 4 * 16 + ((r % 16) ^ (2 * j))) * 16 + kq % 4 * 4);
  }
  // this lane's group of 16 weights of 8 columns, of NT such: column lane / 8 of the wave's
  // 8 columns i
  const int8_t *q[NT];
  int kw[NT];
#pragma unroll
  for (int i = 0; i < NT; i++) {
    const int col = (wave * NT + i) * 8 + lane / 8;
    q[i] = g.q + size_t(min(n0 + col, g.N - 1)) * g.ldq;
    kw[i] = 16 * ((lane % 8) ^ q8_turn(col % 16));
  }
  uint32_t from[2], fromw[2];
#pragma unroll
  for (int o = 0; o < 2; o++) {
    from[o] = uint32_t((o * 64 + lg * 16 + (li ^ (2 * (4 * o + lg)))) * 16 + wm * MT * 2048);
    fromw[o] = uint32_t(WORDS + wn * NT * 2048 + li * 128 + ((4 * o + lg) ^ q8_turn(li)) * 16);
  }

  v4i_t acc[MT][NP][NT] = {};
  T w[QUADS][4];
  auto load_words = [&](int s) __attribute__((always_inline)) {  // of a step within K
#pragma unroll
    for (int i = 0; i < QUADS; i++) __builtin_memcpy(w[i], a[i] + (128 * s + 4 * kq), sizeof w[i]);
  };
  auto load_last = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QUADS; i++) load4<T>(a[i], 128 * s + 4 * kq, g.K, w[i]);
  };
  auto load_weights = [&](int s, uint8_t *buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; i++)  // past the end of a row they meet words' zeros
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void *)(q[i] + min(128 * s + kw[i], end)),
          (__attribute__((address_space(3))) void *)(buf + WORDS + (wave * NT + i) * 1024), 16, 0, 0);
  };
  auto put = [&](uint8_t *buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QUADS; i++) {
      uint32_t d[NP];
      planes4<T>(w[i], d);
#pragma unroll
      for (int p = 0; p < NP; p++) *reinterpret_cast<uint32_t *>(buf + p * PLANE + to[i]) = d[p];
    }
  };
  // this wave's LDS accesses are done, its loads into LDS (which the compiler does not wait
  // for) among them, and every wave's
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  auto compute = [&](const uint8_t *buf) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 0; o < 2; o++) {
      v4i_t b[NT];
#pragma unroll
      for (int t = 0; t < NT; t++) b[t] = *reinterpret_cast<const v4i_t *>(buf + fromw[o] + t * 2048);
#pragma unroll
      for (int p = 0; p < NP; p++)
#pragma unroll
        for (int i = 0; i < MT; i++) {
          const v4i_t d = *reinterpret_cast<const v4i_t *>(buf + p * PLANE + i * 2048 + from[o]);
#pragma unroll
          for (int t = 0; t < NT; t++) acc[i][p][t] = mfma64(d, b[t], acc[i][p][t]);
        }
    }
  };
  // Steps within K have no branch between a load and its use (at a join the compiler waits
  // for all of them); a last step past K is loaded word by word.
  const int whole = min(s1, g.K / 128);
  load_weights(s0, lds[0]);
  if (s0 < whole) load_words(s0);
  else load_last(s0);
  put(lds[0]);
  barrier();
  int s = s0;
  for (; s + 1 < whole; s++) {
    uint8_t *buf = lds[(s - s0) & 1], *next = lds[(s + 1 - s0) & 1];
    load_words(s + 1);
    load_weights(s + 1, next);
    __builtin_amdgcn_sched_barrier(0);  // asked for here, not where they are used
    compute(buf);
    __builtin_amdgcn_sched_barrier(0);
    put(next);
    barrier();
  }
  if (s + 1 < s1) {
    uint8_t *buf = lds[(s - s0) & 1], *next = lds[(s + 1 - s0) & 1];
    load_weights(s + 1, next);
    load_last(s + 1);
    compute(buf);
    put(next);
    barrier();
    s++;
  }
  compute(lds[(s - s0) & 1]);

  int32_t sn[NT], sm[MT][4];
#pragma unroll
  for (int t = 0; t < NT; t++) sn[t] = g.scale ? g.scale[min(n0 + (wn * NT + t) * 16 + li, g.N - 1)] : 1;
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) sm[i][r] = g.tok ? g.tok[min(m0 + (wm * MT + i) * 16 + 4 * lg + r, g.M - 1)] : 1;
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int m = m0 + (wm * MT + i) * 16 + 4 * lg + r;
      if (m >= g.M) continue;
      T *c = g.c + size_t(m) * g.ldc;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const int n = n0 + (wn * NT + t) * 16 + li;
        T v = 0;
#pragma unroll
        for (int p = 0; p < NP; p++) v += plane_word<T>(acc[i][p][t][r], p);
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

template <typename T>
hipError_t launch_part(const Launch &L, const Q8Args<T> &g) {
  constexpr int NP = int(sizeof(T));
  if (g.M <= 16) {
    const int steps = (g.K + 127) / 128, waves = std::min(steps, 16);
    const dim3 grid(unsigned((g.N + 15) / 16)), block(64u * unsigned(waves));
    if (g.M <= 16 / NP) hipLaunchKernelGGL((k_q8_few<T, true>), grid, block, 0, L.stream, g);
    else hipLaunchKernelGGL((k_q8_few<T, false>), grid, block, 0, L.stream, g);
    return hipGetLastError();
  }
  const int steps = (g.K + 127) / 128, exact = (steps + kExact / 128 - 1) / (kExact / 128);
  auto many = [&](auto mt, auto nt) {
    constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value;
    const int rows = (g.M + 32 * MT - 1) / (32 * MT), cols = (g.N + 64 * NT - 1) / (64 * NT);
    const size_t tiles = size_t(rows) * size_t(cols);
    // K is split where the tiles leave CUs without work, into no fewer than four steps
    const int fill = int(std::min<size_t>(size_t(std::max(steps / 4, 1)), std::max<size_t>(size_t(L.num_cu) / tiles, 1)));
    const int splits = std::max(exact, fill);
    if (tiles * size_t(splits) > kMostThreads / 512) return hipErrorInvalidValue;  // more memory than there is
    if (splits > 1) {
      const size_t want = (size_t(g.M) * size_t(g.N) + 255) / 256;
      hipLaunchKernelGGL((k_q8_clear<T>), dim3(unsigned(std::min(want, size_t(L.num_cu) * 8))), dim3(256), 0, L.stream, g);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((k_q8_many<T, MT, NT>), dim3(unsigned(tiles * size_t(splits))), dim3(512), 0, L.stream, g, rows, cols,
                       splits);
    return hipGetLastError();
  };
  auto wide = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    const size_t rows = size_t(g.M + 32 * MT - 1) / (32 * MT), cu = size_t(L.num_cu);
    auto tiles = [&](int nt) { return rows * (size_t(g.N) + 64 * nt - 1) / (64 * nt); };
    if (tiles(4) >= cu) return many(mt, std::integral_constant<int, 4>{});
    if (tiles(3) >= cu) return many(mt, std::integral_constant<int, 3>{});
    if (tiles(2) >= cu) return many(mt, std::integral_constant<int, 2>{});
    return many(mt, std::integral_constant<int, 1>{});
  };
  if constexpr (NP == 4)
    if (g.M > 32) return wide(std::integral_constant<int, 2>{});
  return wide(std::integral_constant<int, 1>{});
}

}  // namespace

template <typename T>
hipError_t launch_gemm_q8(const Launch &L, const Q8Args<T> &g) {
  if (g.K > kQ8MaxK) return hipErrorInvalidValue;
  // HIP cuts a launch of 2^32 threads along a dimension short: in parts of at most 2^16
  // rows by 2^14 columns, 2^11 by 2^8 tiles of 512 threads, and K in up to 2^8 parts, the
  // grid stays below that
  constexpr int rows = 1 << 16, cols = 1 << 14;
  for (int64_t m = 0; m < g.M; m += rows)
    for (int64_t n = 0; n < g.N; n += cols) {
      Q8Args<T> p = g;
      p.M = int(std::min<int64_t>(g.M - m, rows));
      p.N = int(std::min<int64_t>(g.N - n, cols));
      p.a += size_t(m) * g.lda;
      p.q += size_t(n) * g.ldq;
      if (p.scale) p.scale += n;
      if (p.tok) p.tok += m;
      p.c += size_t(m) * g.ldc + size_t(n);
      const hipError_t e = launch_part<T>(L, p);
      if (e != hipSuccess) return e;
    }
  return hipSuccess;
}
template hipError_t launch_gemm_q8<uint32_t>(const Launch &, const Q8Args<uint32_t> &);
template hipError_t launch_gemm_q8<uint64_t>(const Launch &, const Q8Args<uint64_t> &);

}  // namespace mpcx
