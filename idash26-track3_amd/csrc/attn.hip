// attn.hip -- the paged cache of masked keys and values, and the attention
// products that read it (Beaver gates of both parties).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn.h"
#include "digits.h"
#include "launch_util.h"

namespace mpcx {

// ---------------------------------------------------------------------------
// Rows into the cache: workgroup row y = plane, one thread per pair of words.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void k_cache_append(AppendArgs<T> g) {
  const int p = int(blockIdx.y);
  const T *rows = g.rows[p];
  T *pool = g.pool[p];
  const bool rot = g.rotate[p];
  const size_t row = size_t(g.c.heads) * g.c.dim, n = g.n_tok * row;
  for (size_t e = size_t(blockIdx.x) * 256 + threadIdx.x; e < n; e += size_t(gridDim.x) * 256) {
    const size_t t = e / row;
    const int h = int(e % row) / g.c.dim, i = int(e % row) % g.c.dim;
    const int64_t slot = g.slot[t];
    if (slot < 0 || slot >= g.c.n_pages * g.c.page) continue;
    const T *x = rows + t * g.ld[p] + size_t(h) * g.c.dim;
    T v = x[i];
    if (rot) {
      const int at = g.pos[t];
      if (at < 0 || at >= g.n_pos) continue;
      if (i >= 2 * g.half) {
        v <<= g.shift;
      } else {
        const bool second = g.pairs ? (i & 1) : i >= g.half;
        const int f = g.pairs ? i >> 1 : (second ? i - g.half : i);
        const T c = g.cos[size_t(at) * g.half + f], s = g.sin[size_t(at) * g.half + f];
        const T o = x[g.pairs ? i ^ 1 : (second ? i - g.half : i + g.half)];
        v = second ? T(s * o + c * v) : T(c * v - s * o);
      }
    }
    const size_t page = size_t(slot / g.c.page), in = size_t(slot % g.c.page);
    pool[((page * g.c.heads + h) * g.c.page + in) * g.c.dim + i] = v;
  }
}

template <typename T>
hipError_t launch_cache_append(const Launch &L, const AppendArgs<T> &g) {
  const size_t n = g.n_tok * g.c.heads * g.c.dim;
  const size_t want = (n + 255) / 256, cap = size_t(L.num_cu) * 64;
  hipLaunchKernelGGL(k_cache_append<T>, dim3(unsigned(want < cap ? want : cap), unsigned(g.n_planes)), dim3(256), 0,
                     L.stream, g);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// attention products
// ---------------------------------------------------------------------------
// What token t sees: keys [lo, hi) and the first word of its block of scores.
// Ranges and blocks that do not lie inside the bounds see nothing.
struct TokenRange {
  int lo, hi;
  int64_t off;
};
__device__ __forceinline__ TokenRange token_range(const AttnDims &d, int t) {
  TokenRange r;
  r.lo = d.lo[t];
  r.hi = d.hi[t];
  r.off = d.off[t];
  const int64_t n = int64_t(r.hi) - r.lo;
  if (r.lo < 0 || n <= 0 || r.hi > int64_t(d.max_pages) * d.c.page || r.off < 0 || r.off > d.n_scores ||
      n * d.heads > d.n_scores - r.off)
    r.lo = r.hi = 0, r.off = 0;
  return r;
}
// Row `key` (inside the page row) of sequence b's kv head in a cache plane: its first
// word, and whether its page is in the cache (else the word is page 0's).  Loads of
// rows have no branches around them, so that many are in flight: a row that does not
// exist is read at a place that does, and its products are left out.
struct CacheRow {
  int64_t at;
  bool in;
};
__device__ __forceinline__ CacheRow cache_row(const AttnDims &d, int b, int head, int key) {
  const uint32_t page = uint32_t(key) / uint32_t(d.c.page), slot = uint32_t(key) - page * uint32_t(d.c.page);
  const int p = d.pages[int64_t(b) * d.max_pages + page];
  CacheRow r;
  r.in = p >= 0 && p < d.c.n_pages;
  r.at = ((int64_t(r.in ? p : 0) * d.c.heads + head) * d.c.page + slot) * d.c.dim;
  return r;
}

// The products of a form, as terms X_t Y_t of a left and a right word (words of the
// planes that a form does not use are not loaded):
//   BOTH  (x - a0)(y - b0), (-x) b1, (-a1) y;  P0 and P1 the party's part of these;
//   DEAL  x b1, a1 b0
template <AttnForm F>
struct Form {
  static constexpr bool both = F == AttnForm::BOTH, p0 = F == AttnForm::P0, deal = F == AttnForm::DEAL;
  static constexpr int terms = both ? 3 : p0 ? 1 : 2;
  static constexpr bool a0 = both || p0, a1 = !p0, y = !deal, b0 = F != AttnForm::P1, b1 = !p0;
};
// balanced digits of term t's left words of a 16-byte group
template <AttnForm F, typename T>
__device__ __forceinline__ uint4 left_digits(int t, uint4 x, uint4 a0, uint4 a1) {
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (F == AttnForm::DEAL) return t == 0 ? wide_digits<T>(x, z) : wide_digits<T>(a1, z);
  if constexpr (F == AttnForm::P0) return wide_digits<T>(x, a0);
  if constexpr (F == AttnForm::P1) return t == 0 ? wide_digits<T>(z, x) : wide_digits<T>(z, a1);
  return t == 0 ? wide_digits<T>(x, a0) : t == 1 ? wide_digits<T>(z, x) : wide_digits<T>(z, a1);
}
template <AttnForm F, typename T>
__device__ __forceinline__ uint4 right_digits(int t, uint4 y, uint4 b0, uint4 b1) {
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (F == AttnForm::DEAL) return t == 0 ? wide_digits<T>(b1, z) : wide_digits<T>(b0, z);
  if constexpr (F == AttnForm::P0) return wide_digits<T>(y, b0);
  if constexpr (F == AttnForm::P1) return t == 0 ? wide_digits<T>(b1, z) : wide_digits<T>(y, z);
  return t == 0 ? wide_digits<T>(y, b0) : t == 1 ? wide_digits<T>(b1, z) : wide_digits<T>(y, z);
}
template <AttnForm F, typename T>
__device__ __forceinline__ T attn_start(const AttnArgs<T> &g, size_t i) {
  if constexpr (F == AttnForm::P1) return g.c1[i];
  if constexpr (F == AttnForm::BOTH) return g.c0[i] + g.c1[i];
  return g.c0[i];
}
// the 16-byte group of words [i, i + 16 / sizeof(T)) of a row of n words at p (VEC:
// whole groups, 16-byte aligned rows), some words of the row past its end
template <typename T, bool VEC>
__device__ __forceinline__ uint4 row_group(const T *p, int i, int n) {
  constexpr int G = 16 / int(sizeof(T));
  uint4 v;
  if constexpr (VEC) {
    v = *reinterpret_cast<const uint4 *>(p + (i < n ? i : 0));
  } else {
    T w[G];
#pragma unroll
    for (int e = 0; e < G; e++) w[e] = p[min(i + e, n - 1)];
    __builtin_memcpy(&v, w, 16);
  }
  return v;
}
// the words of a group that lie past n words (or all: !in) set to zero
template <typename T>
__device__ __forceinline__ uint4 group_mask(uint4 v, int i, int n, bool in) {
  constexpr int G = 16 / int(sizeof(T));
  T w[G];
  __builtin_memcpy(w, &v, 16);
#pragma unroll
  for (int e = 0; e < G; e++) w[e] = in && i + e < n ? w[e] : T(0);
  __builtin_memcpy(&v, w, 16);
  return v;
}
template <typename T>
__device__ __forceinline__ v4i_t v4(uint4 v) {
  return v4i_t{int(v.x), int(v.y), int(v.z), int(v.w)};
}

// A tile is 16 rows (token, query head) of one sequence that read one head of the
// cache.  What its rows see, by lane li of the first 16 threads into LDS:
struct TileRows {
  int lo[16], hi[16];
  int64_t base[16];  // key j's score is word base + j
  int64_t row[16];   // (token heads + head): the row of queries and outputs, -1: no row
  int tok[16], head[16];
  int klo, khi;  // all keys the rows see lie in [klo, khi)
};
__device__ __forceinline__ void tile_rows(const AttnDims &d, int b, int kv, int64_t e0, TileRows &s) {
  const int tid = int(threadIdx.x), m = d.heads / d.c.heads;
  if (tid < 16) {
    const int t0 = max(d.qstart[b], 0), t1 = min(d.qstart[b + 1], d.n_tok);
    const int64_t e = e0 + tid;
    const int64_t t = t0 + e / m;
    TokenRange r = {0, 0, 0};
    int64_t row = -1;
    const int head = kv * m + int(e % m);
    if (t < t1) {
      r = token_range(d, int(t));
      row = t * d.heads + head;
    }
    s.lo[tid] = r.lo;
    s.hi[tid] = r.hi;
    s.base[tid] = r.off + int64_t(head) * (r.hi - r.lo) - r.lo;
    s.row[tid] = row;
    s.tok[tid] = int(t);
    s.head[tid] = head;
    int lo = r.hi > r.lo ? r.lo : INT32_MAX, hi = r.hi;
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) {
      lo = min(lo, __shfl_xor(lo, k, 16));
      hi = max(hi, __shfl_xor(hi, k, 16));
    }
    s.klo = hi > 0 ? lo : 0;
    s.khi = hi;
  }
}
// A launch's units of work: pair (sequence, cache head) slowest, then tile of rows,
// column group (mix) and key split; a unit strides over tiles by `tiles` and over
// keys by `splits`, so the hints they come from do not bound what is computed.
struct Units {
  int64_t n = 0;
  int tiles = 1, cols = 1, splits = 1;
};
struct Unit {
  int b, kv, tile, col, split;
};
__device__ __forceinline__ Unit unit_of(const AttnDims &d, const Units &n, int64_t u) {
  Unit r;
  r.split = int(u % n.splits);
  u /= n.splits;
  r.col = int(u % n.cols);
  u /= n.cols;
  r.tile = int(u % n.tiles);
  u /= n.tiles;
  r.kv = int(u % d.c.heads);
  r.b = int(u / d.c.heads);
  return r;
}

// ---------------------------------------------------------------------------
// Scores.  A workgroup holds a tile's queries in LDS as digits, one plane per term;
// each of its four waves takes 16 keys at a time, whose rows go from memory straight
// to the lanes that feed them to the matrix cores (lane (li, lg): key li, 16-byte
// group lg of every 64 bytes).
// ---------------------------------------------------------------------------
constexpr int kScoreWaves = 4, kScoreKeys = 16 * kScoreWaves;
template <AttnForm F, typename T, bool VEC>
__global__ __launch_bounds__(64 * kScoreWaves) void k_attn_scores(AttnArgs<T> g, Units units, int slab) {
  constexpr int G = 16 / int(sizeof(T)), NQ = int(sizeof(T)), NT = Form<F>::terms, CB = 4;
  extern __shared__ __align__(16) uint4 xs[];  // [term][16][groups of the slab + 1]
  __shared__ TileRows rows;
  const AttnDims &d = g.d;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
  const int sg = slab / G + 1;  // groups of an LDS row
  const int slabs = (d.c.dim + slab - 1) / slab;
  const uint4 z4 = make_uint4(0u, 0u, 0u, 0u);
  auto stage = [&](int s) {
    for (int e = tid; e < 16 * (slab / G); e += 64 * kScoreWaves) {
      const int r = e / (slab / G), q = e % (slab / G), i = s * slab + q * G;
      const bool in = rows.row[r] >= 0;
      const int64_t at = in ? rows.row[r] * d.c.dim : 0;
      auto group = [&](const T *p) { return group_mask<T>(row_group<T, VEC>(p + at, i, d.c.dim), i, d.c.dim, in); };
      const uint4 x = group(g.x), a0 = Form<F>::a0 ? group(g.a0) : z4, a1 = Form<F>::a1 ? group(g.a1) : z4;
#pragma unroll
      for (int t = 0; t < NT; t++) xs[(t * 16 + r) * sg + q] = left_digits<F, T>(t, x, a0, a1);
    }
  };
  for (int64_t w = blockIdx.x; w < units.n; w += gridDim.x) {
    const Unit u = unit_of(d, units, w);
    const int64_t m = d.heads / d.c.heads;
    const int64_t n_rows = int64_t(min(d.qstart[u.b + 1], d.n_tok) - max(d.qstart[u.b], 0)) * m;
    for (int64_t e0 = int64_t(u.tile) * 16; e0 < n_rows; e0 += int64_t(units.tiles) * 16) {
      __syncthreads();
      tile_rows(d, u.b, u.kv, e0, rows);
      __syncthreads();
      if (slabs == 1) {
        stage(0);
        __syncthreads();
      }
      const int khi = rows.khi;
      for (int64_t kb = rows.klo + int64_t(u.split) * kScoreKeys; kb < khi; kb += int64_t(units.splits) * kScoreKeys) {
        const int64_t key = kb + 16 * wave + li;
        const CacheRow j = cache_row(d, u.b, u.kv, int(min(key, int64_t(khi) - 1)));
        T vs[4] = {0, 0, 0, 0};
        for (int s = 0; s < slabs; s++) {
          if (slabs > 1) {
            __syncthreads();
            stage(s);
            __syncthreads();
          }
          v4i_t acc[NQ];
#pragma unroll
          for (int q = 0; q < NQ; q++) acc[q] = v4i_t{0, 0, 0, 0};
          const int words = min(slab, d.c.dim - s * slab), chunks = (words + 4 * G - 1) / (4 * G);
          for (int c0 = 0; c0 < chunks; c0 += CB) {
            uint4 y[CB], b0[CB], b1[CB];
#pragma unroll
            for (int c = 0; c < CB; c++) {
              if (c0 + c >= chunks) break;
              const int i = s * slab + ((c0 + c) * 4 + lg) * G;
              y[c] = Form<F>::y ? row_group<T, VEC>(g.y + j.at, i, d.c.dim) : z4;
              b0[c] = Form<F>::b0 ? row_group<T, VEC>(g.b0 + j.at, i, d.c.dim) : z4;
              b1[c] = Form<F>::b1 ? row_group<T, VEC>(g.b1 + j.at, i, d.c.dim) : z4;
            }
#pragma unroll
            for (int c = 0; c < CB; c++) {
              if (c0 + c >= chunks) break;
#pragma unroll
              for (int t = 0; t < NT; t++) {
                v4i_t as[NQ];
                digit_shifts<T>(xs[(t * 16 + li) * sg + (c0 + c) * 4 + lg], as);
                const v4i_t bv = v4<T>(right_digits<F, T>(t, y[c], b0[c], b1[c]));
#pragma unroll
                for (int q = 0; q < NQ; q++) acc[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(as[q], bv, acc[q], 0, 0, 0);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 4; r++) vs[r] += digit_fold<T>(acc, r);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {  // accumulator register r of lane (li, lg): row 4 lg + r, key li
          const int row = 4 * lg + r;
          if (key < rows.lo[row] || key >= rows.hi[row]) continue;
          const size_t o = size_t(rows.base[row] + key);
          T v = (j.in ? vs[r] : T(0)) + attn_start<F>(g, o);
          if constexpr (F == AttnForm::BOTH || F == AttnForm::P0)
            if (g.slope) v += g.slope[rows.head[row]] * T(key - g.pos[rows.tok[row]]);
          g.out[o] = v;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Weighted sums.  A wave takes 64 bytes of keys at a time (16 or 8): their weights as
// the 16 rows' operand, and 256 bytes of columns of the values' rows, lane (li, lg)
// loading group li of the rows lg G .. + G - 1, so that word q of its groups is the
// operand of column tile q.  The waves of a workgroup and the launch's splits share
// the keys out; their sums meet in LDS and in integer additions to the output, whose
// order does not matter.
// ---------------------------------------------------------------------------
constexpr int kMixWaves = 4;
template <AttnForm F, typename T, bool VEC>
__global__ __launch_bounds__(64 * kMixWaves) void k_attn_mix(AttnArgs<T> g, Units units) {
  constexpr int G = 16 / int(sizeof(T)), NQ = int(sizeof(T)), NT = Form<F>::terms, CK = 4 * G;
  constexpr int kFlush = 4096 / CK;  // chunks whose digit sums stay exact (3 terms, Z_2^64)
  __shared__ TileRows rows;
  __shared__ T red[kMixWaves][G * 4][64];
  const AttnDims &d = g.d;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
  const uint4 z4 = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t w = blockIdx.x; w < units.n; w += gridDim.x) {
    const Unit u = unit_of(d, units, w);
    const int64_t m = d.heads / d.c.heads;
    const int64_t n_rows = int64_t(min(d.qstart[u.b + 1], d.n_tok) - max(d.qstart[u.b], 0)) * m;
    const int col = u.col * 16 * G + li * G;  // this lane's columns
    for (int64_t e0 = int64_t(u.tile) * 16; e0 < n_rows; e0 += int64_t(units.tiles) * 16) {
      __syncthreads();
      tile_rows(d, u.b, u.kv, e0, rows);
      __syncthreads();
      const int khi = rows.khi, lo = rows.lo[li], hi = rows.hi[li];
      const int64_t base = rows.base[li];
      v4i_t acc[G][NQ];
      T vs[G][4];
#pragma unroll
      for (int q = 0; q < G; q++)
#pragma unroll
        for (int r = 0; r < 4; r++) vs[q][r] = 0;
      int64_t kb = rows.klo + (int64_t(u.split) * kMixWaves + wave) * CK;
      const int64_t step = int64_t(units.splits) * kMixWaves * CK;
      while (kb < khi) {
#pragma unroll
        for (int q = 0; q < G; q++)
#pragma unroll
          for (int s = 0; s < NQ; s++) acc[q][s] = v4i_t{0, 0, 0, 0};
        for (int it = 0; it < kFlush && kb < khi; it++, kb += step) {
          const int64_t k0 = kb + lg * G;  // this lane's keys k0 .. k0 + G - 1
          uint4 y[G], b0[G], b1[G];
          CacheRow j[G];
#pragma unroll
          for (int i = 0; i < G; i++) j[i] = cache_row(d, u.b, u.kv, int(min(k0 + i, int64_t(khi) - 1)));
          T xw[G], a0w[G], a1w[G];
          bool in[G];
#pragma unroll
          for (int i = 0; i < G; i++) {
            in[i] = k0 + i >= lo && k0 + i < hi;
            const int64_t o = in[i] ? base + k0 + i : 0;
            xw[i] = g.x[o];
            a0w[i] = Form<F>::a0 ? g.a0[o] : T(0);
            a1w[i] = Form<F>::a1 ? g.a1[o] : T(0);
          }
#pragma unroll
          for (int i = 0; i < G; i++) {
            y[i] = Form<F>::y ? row_group<T, VEC>(g.y + j[i].at, col, d.c.dim) : z4;
            b0[i] = Form<F>::b0 ? row_group<T, VEC>(g.b0 + j[i].at, col, d.c.dim) : z4;
            b1[i] = Form<F>::b1 ? row_group<T, VEC>(g.b1 + j[i].at, col, d.c.dim) : z4;
          }
#pragma unroll
          for (int i = 0; i < G; i++) {  // a weight outside the range, or of a row that is not there: no product
            const bool use = in[i] && j[i].in;
            xw[i] = use ? xw[i] : T(0);
            a0w[i] = use ? a0w[i] : T(0);
            a1w[i] = use ? a1w[i] : T(0);
          }
          uint4 x, a0, a1;
          __builtin_memcpy(&x, xw, 16);
          __builtin_memcpy(&a0, a0w, 16);
          __builtin_memcpy(&a1, a1w, 16);
#pragma unroll
          for (int t = 0; t < NT; t++) {
            v4i_t as[NQ];
            digit_shifts<T>(left_digits<F, T>(t, x, a0, a1), as);
            uint32_t dig[G][4];
#pragma unroll
            for (int i = 0; i < G; i++) {
              const uint4 v = right_digits<F, T>(t, y[i], b0[i], b1[i]);
              dig[i][0] = v.x, dig[i][1] = v.y, dig[i][2] = v.z, dig[i][3] = v.w;
            }
#pragma unroll
            for (int q = 0; q < G; q++) {
              v4i_t bv;
              if constexpr (sizeof(T) == 4) bv = v4i_t{int(dig[0][q]), int(dig[1][q]), int(dig[G - 2][q]), int(dig[G - 1][q])};
              else bv = v4i_t{int(dig[0][2 * q]), int(dig[0][2 * q + 1]), int(dig[1][2 * q]), int(dig[1][2 * q + 1])};
#pragma unroll
              for (int s = 0; s < NQ; s++)
                acc[q][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(as[s], bv, acc[q][s], 0, 0, 0);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < G; q++)
#pragma unroll
          for (int r = 0; r < 4; r++) vs[q][r] += digit_fold<T>(acc[q], r);
      }
#pragma unroll
      for (int q = 0; q < G; q++)
#pragma unroll
        for (int r = 0; r < 4; r++) red[wave][q * 4 + r][lane] = vs[q][r];
      __syncthreads();
      for (int e = tid; e < G * 4 * 64; e += 64 * kMixWaves) {
        // words in the order of the output: row, column (G a lane)
        const int row = e / (16 * G), c = e % (16 * G), q = c % G, l = 16 * (row / 4) + c / G, at = q * 4 + row % 4;
        const int oc = u.col * 16 * G + c;
        if (rows.row[row] < 0 || oc >= d.c.dim) continue;
        T v = 0;
#pragma unroll
        for (int k = 0; k < kMixWaves; k++) v += red[k][at][l];
        const size_t o = size_t(rows.row[row]) * d.c.dim + oc;
        if (units.splits == 1) {
          g.out[o] = v + attn_start<F>(g, o);
        } else if constexpr (sizeof(T) == 4) {
          atomicAdd(reinterpret_cast<unsigned int *>(&g.out[o]), static_cast<unsigned int>(v));
        } else {
          atomicAdd(reinterpret_cast<unsigned long long *>(&g.out[o]), static_cast<unsigned long long>(v));
        }
      }
    }
  }
}
// the product terms, which the splits add to
template <AttnForm F, typename T>
__global__ __launch_bounds__(256) void k_mix_init(AttnArgs<T> g, size_t n) {
  for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += size_t(gridDim.x) * 256)
    g.out[i] = attn_start<F>(g, i);
}

template <typename T>
bool vec_rows(const AttnArgs<T> &g, bool left) {
  bool ok = g.d.c.dim % int(16 / sizeof(T)) == 0;
  for (const void *p : {(const void *)g.y, (const void *)g.b0, (const void *)g.b1})
    ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  if (left)
    for (const void *p : {(const void *)g.x, (const void *)g.a0, (const void *)g.a1})
      ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  return ok;
}
// about `want` units, at least one tile and one split each
Units units_for(const AttnDims &d, int cols, int64_t want, int64_t keys_per_split) {
  Units u;
  u.cols = cols;
  const int64_t m = d.heads / d.c.heads, pairs = int64_t(d.n_seq) * d.c.heads;
  const int64_t tiles = std::min<int64_t>((int64_t(d.max_q) * m + 15) / 16, 1 << 20);
  const int64_t base = pairs * cols * tiles, most = (int64_t(d.max_keys) + keys_per_split - 1) / keys_per_split;
  u.tiles = int(tiles);
  u.splits = int(std::max<int64_t>(1, std::min<int64_t>((want + base - 1) / base, std::min<int64_t>(most, 1 << 16))));
  u.n = base * u.splits;
  return u;
}
unsigned grid_of(const Units &u) { return unsigned(std::min<int64_t>(u.n, 1 << 24)); }

template <AttnForm F, typename T>
hipError_t scores_at(const Launch &L, const AttnArgs<T> &g) {
  constexpr int G = 16 / int(sizeof(T));
  // the tile's queries in at most 64 KB: slabs of whole 64-byte groups
  const int most = 64 * 1024 / (Form<F>::terms * 16 * int(sizeof(T))) / (4 * G) * (4 * G) - 4 * G;
  const int slab = std::min((g.d.c.dim + 4 * G - 1) / (4 * G) * (4 * G), most);
  const size_t lds = size_t(Form<F>::terms) * 16 * (slab / G + 1) * 16;
  const Units u = units_for(g.d, 1, int64_t(L.num_cu) * 8, kScoreKeys);
  if (vec_rows(g, true))
    hipLaunchKernelGGL((k_attn_scores<F, T, true>), dim3(grid_of(u)), dim3(64 * kScoreWaves), lds, L.stream, g, u, slab);
  else
    hipLaunchKernelGGL((k_attn_scores<F, T, false>), dim3(grid_of(u)), dim3(64 * kScoreWaves), lds, L.stream, g, u, slab);
  return hipGetLastError();
}
template <AttnForm F, typename T>
hipError_t mix_at(const Launch &L, const AttnArgs<T> &g) {
  constexpr int G = 16 / int(sizeof(T));
  const Units u =
      units_for(g.d, (g.d.c.dim + 16 * G - 1) / (16 * G), int64_t(L.num_cu) * 4, int64_t(kMixWaves) * 4 * G * 4);
  if (u.splits > 1) {
    const size_t n = size_t(g.d.n_tok) * g.d.heads * g.d.c.dim, want = (n + 255) / 256, cap = size_t(L.num_cu) * 32;
    hipLaunchKernelGGL((k_mix_init<F, T>), dim3(unsigned(want < cap ? want : cap)), dim3(256), 0, L.stream, g, n);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (vec_rows(g, false))
    hipLaunchKernelGGL((k_attn_mix<F, T, true>), dim3(grid_of(u)), dim3(64 * kMixWaves), 0, L.stream, g, u);
  else
    hipLaunchKernelGGL((k_attn_mix<F, T, false>), dim3(grid_of(u)), dim3(64 * kMixWaves), 0, L.stream, g, u);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_attn_scores(const Launch &L, AttnForm form, const AttnArgs<T> &g) {
  switch (form) {
    case AttnForm::BOTH: return scores_at<AttnForm::BOTH, T>(L, g);
    case AttnForm::P0: return scores_at<AttnForm::P0, T>(L, g);
    case AttnForm::P1: return scores_at<AttnForm::P1, T>(L, g);
    case AttnForm::DEAL: return scores_at<AttnForm::DEAL, T>(L, g);
  }
  return hipErrorInvalidValue;
}
template <typename T>
hipError_t launch_attn_mix(const Launch &L, AttnForm form, const AttnArgs<T> &g) {
  switch (form) {
    case AttnForm::BOTH: return mix_at<AttnForm::BOTH, T>(L, g);
    case AttnForm::P0: return mix_at<AttnForm::P0, T>(L, g);
    case AttnForm::P1: return mix_at<AttnForm::P1, T>(L, g);
    case AttnForm::DEAL: return mix_at<AttnForm::DEAL, T>(L, g);
  }
  return hipErrorInvalidValue;
}

#define INST(T)                                                                                       \
  template hipError_t launch_cache_append<T>(const Launch &, const AppendArgs<T> &);                  \
  template hipError_t launch_attn_scores<T>(const Launch &, AttnForm, const AttnArgs<T> &);           \
  template hipError_t launch_attn_mix<T>(const Launch &, AttnForm, const AttnArgs<T> &);
INST(uint32_t)
INST(uint64_t)

}  // namespace mpcx
