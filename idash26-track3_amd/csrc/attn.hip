// attn.hip -- the paged cache of masked keys and values, and the attention
// products that read it (Beaver gates of both parties).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn.h"
#include "digits.h"
#include "launch_util.h"

namespace mpcx {

// ---------------------------------------------------------------------------
// Rows into the cache: one thread per group of G words of a token's row (16 bytes where
// every row and table is aligned to them), one row of workgroups per plane.  A rotated
// word needs its partner too, which the neighbouring thread or one half a rotation away
// reads as its own: the second read is served by the caches.  Bound by the bytes, each
// read and written once: 6000 tokens of 4 heads of 80 in Z_2^64, six planes, 47.7 us, 186
// MB at 3.9 TB/s (a large copy reaches 4.7); word by word 76.5.  A few tokens are bound by
// the launch (48 of 8 heads of 128: 3.7 us).
// ---------------------------------------------------------------------------
template <typename T, int G>
struct Words {
  T w[G];
};
template <typename T, int G>
__device__ __forceinline__ Words<T, G> load_words(const T *p) {
  Words<T, G> r;
  __builtin_memcpy(r.w, __builtin_assume_aligned(p, sizeof(T) * G), sizeof(T) * G);
  return r;
}
template <typename T, int G>
__global__ __launch_bounds__(256) void k_cache_append(AppendArgs<T> g) {
  const int p = int(blockIdx.y);
  const T *rows = g.rows[p];
  T *pool = g.pool[p];
  const size_t ld = g.ld[p];
  const bool rot = g.rotate[p];
  const uint32_t per_head = uint32_t(g.c.dim) / G, row = per_head * uint32_t(g.c.heads);
  const uint64_t slots = uint64_t(g.c.n_pages) * uint64_t(g.c.page);
  // this thread's place (token, group of the row), and the grid's stride as one
  const size_t first = size_t(blockIdx.x) * 256 + threadIdx.x, stride = size_t(gridDim.x) * 256;
  size_t t = first / row;
  uint32_t r = uint32_t(first - t * row);
  const size_t step_t = stride / row;
  const uint32_t step_r = uint32_t(stride - step_t * row);
  for (; t < g.n_tok; t += step_t, r += step_r) {
    if (r >= row) {
      r -= row;
      if (++t >= g.n_tok) break;
    }
    const uint64_t slot = uint64_t(g.slot[t]);
    if (slot >= slots) continue;  // a negative slot, too
    const uint32_t h = r / per_head;
    const int i = int(r - h * per_head) * G;
    const T *x = rows + t * ld + size_t(h) * g.c.dim;
    Words<T, G> v = load_words<T, G>(x + i);
    if (rot) {
      const int at = g.pos[t];
      if (at < 0 || at >= g.n_pos) continue;
      const T *ct = g.cos + size_t(at) * g.half, *st = g.sin + size_t(at) * g.half;
      if (i >= 2 * g.half) {
#pragma unroll
        for (int k = 0; k < G; k++) v.w[k] <<= g.shift;
      } else if (g.pairs) {
        if constexpr (G == 1) {
          const T o = x[i ^ 1], c = ct[i / 2], s = st[i / 2];
          v.w[0] = i & 1 ? T(s * o + c * v.w[0]) : T(c * v.w[0] - s * o);
        } else {
          const Words<T, G / 2> c = load_words<T, G / 2>(ct + i / 2), s = load_words<T, G / 2>(st + i / 2);
#pragma unroll
          for (int k = 0; k < G; k += 2) {
            const T a = v.w[k], b = v.w[k + 1];
            v.w[k] = c.w[k / 2] * a - s.w[k / 2] * b;
            v.w[k + 1] = s.w[k / 2] * a + c.w[k / 2] * b;
          }
        }
      } else {
        const bool second = i >= g.half;
        const int f = second ? i - g.half : i;
        const Words<T, G> c = load_words<T, G>(ct + f), s = load_words<T, G>(st + f);
        const Words<T, G> o = load_words<T, G>(x + (second ? f : f + g.half));
#pragma unroll
        for (int k = 0; k < G; k++)
          v.w[k] = second ? T(s.w[k] * o.w[k] + c.w[k] * v.w[k]) : T(c.w[k] * v.w[k] - s.w[k] * o.w[k]);
      }
    }
    const uint64_t page = slots >> 32 ? slot / uint64_t(g.c.page) : uint64_t(uint32_t(slot) / uint32_t(g.c.page));
    const uint64_t in = slot - page * uint64_t(g.c.page);
    T *to = pool + ((page * g.c.heads + h) * g.c.page + in) * g.c.dim + i;
    __builtin_memcpy(__builtin_assume_aligned(to, sizeof(T) * G), v.w, sizeof(T) * G);
  }
}

template <typename T, int G>
hipError_t append_at(const Launch &L, const AppendArgs<T> &g) {
  const size_t n = g.n_tok * size_t(g.c.heads) * (size_t(g.c.dim) / G);
  const size_t want = (n + 255) / 256, cap = size_t(L.num_cu) * 32;
  hipLaunchKernelGGL((k_cache_append<T, G>), dim3(unsigned(want < cap ? want : cap), unsigned(g.n_planes)), dim3(256), 0,
                     L.stream, g);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_cache_append(const Launch &L, const AppendArgs<T> &g) {
  constexpr int G = 16 / int(sizeof(T));
  bool vec = g.c.dim % G == 0;
  auto check = [&](const void *p) { vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  bool rot = false;
  for (int p = 0; p < g.n_planes; p++) {
    check(g.rows[p]);
    check(g.pool[p]);
    vec = vec && g.ld[p] % G == 0;
    rot = rot || g.rotate[p];
  }
  if (rot) {  // a table row starts at a whole group, or half of one
    vec = vec && g.half % (g.pairs ? G / 2 : G) == 0;
    check(g.cos);
    check(g.sin);
  }
  return vec ? append_at<T, G>(L, g) : append_at<T, 1>(L, g);
}

// ---------------------------------------------------------------------------
// attention products
// ---------------------------------------------------------------------------
// What a token sees: keys [lo, hi) and the first word of its block of scores.
// Ranges and blocks that do not lie inside the bounds see nothing (0, 0, 0).
struct TokenRange {
  int lo, hi;
  int64_t off;
};
__device__ __forceinline__ TokenRange token_range(const AttnDims &d, int t) {
  TokenRange r;
  r.lo = d.lo[t];
  r.hi = d.hi[t];
  r.off = d.off[t];
  const int64_t n = int64_t(r.hi) - r.lo;  // below 2^32, times heads below 2^63
  const bool ok = (r.lo >= 0) & (n > 0) & (r.hi <= int64_t(d.max_pages) * d.c.page) & (r.off >= 0) &
                  (r.off <= d.n_scores) & (n * d.heads <= d.n_scores - r.off);
  r.lo = ok ? r.lo : 0;
  r.hi = ok ? r.hi : 0;
  r.off = ok ? r.off : 0;
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

// Row e of a sequence and a head of the cache is query head e % m of token e / m (m query
// heads a cache head, below 2^31 rows); a tile is 16 of them.  What a row sees:
struct TileRow {
  int lo, hi;
  int64_t base;  // key j's score is word base + j
  int tok, head;
};
__device__ __forceinline__ TileRow tile_row(const AttnDims &d, int t0, int t1, int kv, uint32_t m, uint32_t e) {
  TileRow s;
  const uint32_t q = e / m;
  const bool in = int64_t(t0) + q < t1;
  s.head = kv * int(m) + int(e - q * m);
  s.tok = in ? t0 + int(q) : t0;
  const TokenRange r = token_range(d, s.tok);
  s.lo = in ? r.lo : 0;
  s.hi = in ? r.hi : 0;
  s.base = r.off + int64_t(s.head) * (r.hi - r.lo) - r.lo;
  return s;
}
// smallest lo and largest hi of the rows that see something, over N lanes (hi = 0: none)
template <int N>
__device__ __forceinline__ void tile_keys(const TileRow &s, int &klo, int &khi) {
  int lo = s.hi > s.lo ? s.lo : INT32_MAX, hi = s.hi;
#pragma unroll
  for (int k = 1; k < N; k <<= 1) {
    lo = min(lo, __shfl_xor(lo, k, N));
    hi = max(hi, __shfl_xor(hi, k, N));
  }
  klo = __builtin_amdgcn_readfirstlane(lo);
  khi = __builtin_amdgcn_readfirstlane(hi);
}
// A launch's units of work: pair (sequence, cache head) slowest, then tile of rows,
// column group (mix) and key split: a unit strides over tiles by `tiles` and over keys by
// `splits` steps of its waves, so the hints that these come from do not bound what is
// computed, and a short sequence's units have as much less to do each.  Neighbouring
// units run on different XCDs: an XCD that held whole sequences would be late with the
// longest.
struct Units {
  int n = 0, tiles = 1, cols = 1, splits = 1;
};
// The steps of `step` keys that wave `wave` of a unit takes, from key `at` on (khi: none
// are left).
struct KeySteps {
  int64_t at, stride;
  int khi;
  __device__ __forceinline__ KeySteps(const Units &n, int split, int klo, int khi_, int wave, int waves, int step)
      : at(int64_t(klo) + (int64_t(split) * waves + wave) * step), stride(int64_t(n.splits) * waves * step), khi(khi_) {}
  __device__ __forceinline__ void advance() { at += stride; }
  __device__ __forceinline__ bool any() const { return at < khi; }
};
struct Unit {
  int b, kv, tile, col, split;
};
__device__ __forceinline__ Unit unit_of(const AttnDims &d, const Units &n) {
  Unit r;
  uint32_t u = blockIdx.x;
  r.split = int(u % uint32_t(n.splits));
  u /= uint32_t(n.splits);
  r.col = int(u % uint32_t(n.cols));
  u /= uint32_t(n.cols);
  r.tile = int(u % uint32_t(n.tiles));
  u /= uint32_t(n.tiles);
  r.kv = int(u % uint32_t(d.c.heads));
  r.b = int(u / uint32_t(d.c.heads));
  return r;
}

// Bytes of four ring words by digit: o[p] holds digit p of the words (Z_2^32: digits 0..3
// of the words w; the two halves of Z_2^64 words are digits 0..3 and 4..7).
__device__ __forceinline__ void digit_planes(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&o)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w1, w0, 0x05010400u), b = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(w3, w2, 0x05010400u), d = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
  o[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  o[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  o[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  o[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}
// The same of whole words as 16-byte groups of digits: one group of Z_2^32, two of Z_2^64
template <typename T>
__device__ __forceinline__ void group_planes(uint4 u, uint4 v, uint32_t (&o)[sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    digit_planes(u.x, u.y, u.z, u.w, o);
  } else {
    uint32_t lo[4], hi[4];
    digit_planes(u.x, u.z, v.x, v.z, lo);
    digit_planes(u.y, u.w, v.y, v.w, hi);
#pragma unroll
    for (int p = 0; p < 4; p++) o[p] = lo[p], o[4 + p] = hi[p];
  }
}

// ---------------------------------------------------------------------------
// Scores.  Digits by plane: a 64-word step of the product is bw / 8 planes of 16 bytes
// a lane on either side, and sum_{p + q < bw / 8} 2^(8(p + q)) A_p B_q takes 10 (Z_2^32)
// or 36 (Z_2^64) MFMAs.  A workgroup holds the planes of RT tiles of queries in LDS;
// each of its waves takes 16 keys at a time, whose rows go from memory to the lanes that
// feed them to the matrix cores: lane (li, lg) holds of key li the 16-byte groups 4 c + lg
// (c: the row's 64-byte chunks), so every load reads 64 bytes of each row.  A step's rows
// and the words its products are added to are asked for as soon as the last step's are
// used up, the first ones before the queries are staged, and the page numbers of the
// next keys one tile ahead: no load waits for another.  The words of a launch are dims
// [k0, k0 + kn) of the heads, as many as LDS holds of the queries; `more`: the sums so
// far are in out.
// One token a sequence is bound by the cache's bytes: 8 sequences of up to 4096 keys, 8
// cache heads of 128 in Z_2^32: 77 us a call for 296 MB, 3.8 TB/s (the start, some 10 us
// from the first page number to the first product, and the longest sequence's end are what
// is left); in Z_2^64 226 us for 592 MB, 2.6 TB/s, one party's message 97: at 344 registers
// a wave of the form of both parties runs alone on its SIMD.
// Prompts are bound by the order of work in the waves of the longest rows: 4 x 512 tokens,
// 8 heads of 64 in Z_2^32, 45.4 us a call.  All their workgroups run at once, two waves a
// SIMD, so the launch ends with the waves that take eight steps of 16 keys, while the mean is
// 3.3: over the launch vector instructions issue 15% of the time (2083 a wave, most of them
// the digits') and MFMAs are busy 6% (198 a wave).  A step is some 630 vector instructions
// and 60 MFMAs a wave, 2.9 us of issue for the two waves of a SIMD; the rest of its 4 to 5 us
// they wait for one another, LDS and the rows (asked for before the products instead of
// after them: no faster).
// Four waves, so that one workgroup's start runs beside another's products: calls in
// Z_2^32 by eight take 51.2 us for 4 x 256 tokens against 1024 keys, by four 41.9; 60.7 for
// 3 x 400 of 16 heads of 128, by four 53.2; but 40.4 for the 4 x 512, by four 45.4.  In
// Z_2^64 eight spill: 200 us for the 4 x 512, by four 108.
// ---------------------------------------------------------------------------
constexpr int kScoreWaves = 4;
template <AttnForm F, typename T, bool VEC, int RT>
__global__ __launch_bounds__(64 * kScoreWaves, sizeof(T) == 4 ? 2 : 1) void k_attn_scores(AttnArgs<T> g, Units units,
                                                                                          int k0, int kn, bool more) {
  constexpr int G = 16 / int(sizeof(T)), NQ = int(sizeof(T)), NT = Form<F>::terms;
  constexpr int CH = int(sizeof(T)), PAIR = CH / 4;  // chunks of a step; those of four words
  constexpr bool bias = F == AttnForm::BOTH || F == AttnForm::P0;
  extern __shared__ __align__(16) uint4 xs[];  // [tile][step][term][plane][lane]
  __shared__ int rlo[16 * RT], rhi[16 * RT], rpos[16 * RT];
  __shared__ int slo[16 * RT], shi[16 * RT];
  __shared__ int64_t rbase[16 * RT], sbase[16 * RT];
  __shared__ T rslope[16 * RT];
  const AttnDims &d = g.d;
  const int tid = int(threadIdx.x), lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int steps = (kn + 63) / 64, kend = k0 + kn;
  const uint4 z4 = make_uint4(0u, 0u, 0u, 0u);
  const Unit u = unit_of(d, units);
  const uint32_t m = uint32_t(d.heads) / uint32_t(d.c.heads);
  const int t0 = max(d.qstart[u.b], 0), t1 = min(d.qstart[u.b + 1], d.n_tok);
  const uint32_t n_rows = t1 > t0 ? uint32_t(t1 - t0) * m : 0u;
  const int32_t *table = d.pages + int64_t(u.b) * d.max_pages;
  const uint32_t psize = uint32_t(d.c.page);

  struct Query {
    uint4 x[PAIR], a0[PAIR], a1[PAIR];
  };
  // a step of 16 keys' rows, and what their products are added to
  uint4 y[CH], b0[CH], b1[CH];
  T c0[RT][4], c1[RT][4];
  int64_t kb = 0, at = 0;  // the keys, this lane's key's row
  int step = 0;
  bool in = false;  // its page is in the cache
  v4i_t acc[RT][NQ];
  for (int64_t eb = int64_t(u.tile) * (16 * RT); eb < n_rows; eb += int64_t(units.tiles) * (16 * RT)) {
    const uint32_t e0 = uint32_t(eb);
    // Queries, four words of a row at a time: lane group l's dword c of step s is words of
    // chunk c (Z_2^32) or of chunks 2 c, 2 c + 1 (Z_2^64).  The first are asked for
    // before anything else.
    auto get = [&](int e, Query &q) {
      const int r = e % (16 * RT), l = e / (16 * RT) % 4, c = e / (64 * RT) % 4, s = e / (256 * RT);
      const int i = k0 + 64 * s + 16 * c + l * G;
      const uint32_t qr = e0 + uint32_t(r), qt = qr < n_rows ? qr / m : 0u;
      const bool there = qr < n_rows;
      const int64_t row = (int64_t(t0 + int(qt)) * d.heads + u.kv * int64_t(m) + (there ? qr - qt * m : 0u)) * d.c.dim;
#pragma unroll
      for (int h = 0; h < PAIR; h++) {
        auto group = [&](const T *p) {
          return group_mask<T>(row_group<T, VEC>(p + row, i + 4 * G * h, d.c.dim), i + 4 * G * h, kend, there);
        };
        q.x[h] = group(g.x);
        q.a0[h] = Form<F>::a0 ? group(g.a0) : z4;
        q.a1[h] = Form<F>::a1 ? group(g.a1) : z4;
      }
    };
    auto put = [&](int e, const Query &q) {
      const int r = e % (16 * RT), l = e / (16 * RT) % 4, c = e / (64 * RT) % 4, s = e / (256 * RT);
      if (s >= steps) return;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        uint32_t o[NQ];
        group_planes<T>(left_digits<F, T>(t, q.x[0], q.a0[0], q.a1[0]),
                        left_digits<F, T>(t, q.x[PAIR - 1], q.a0[PAIR - 1], q.a1[PAIR - 1]), o);
        uint32_t *to = reinterpret_cast<uint32_t *>(
            xs + (size_t(r / 16 * steps + s) * NT + t) * NQ * 64 + 16 * l + r % 16);
#pragma unroll
        for (int p = 0; p < NQ; p++) to[p * 256 + c] = o[p];
      }
    };
    Query first;
    get(tid, first);
    const TileRow mine = tile_row(d, t0, t1, u.kv, m, e0 + uint32_t(lane % (16 * RT)));
    int klo, khi;
    tile_keys<16 * RT>(mine, klo, khi);
    KeySteps ahead(units, u.split, klo, khi, wave, kScoreWaves, 16);  // the tile after the one asked for
    const int last = khi > 0 ? khi - 1 : 0;  // keys past the range read the last one's row
    auto page_of = [&](int64_t kb) {
      const uint32_t key = min(uint32_t(kb) + uint32_t(li), uint32_t(last));
      return table[min(key / psize, uint32_t(d.max_pages - 1))];
    };
    __syncthreads();  // the last tile's queries and rows are done with
    if (tid < 16 * RT) {
      rlo[tid] = mine.lo;
      rhi[tid] = mine.hi;
      rbase[tid] = mine.base;
      // where a word is read for a row and key without one: some word of a row that has
      // (a place that others read too, not one that all the GPU reads)
      const uint64_t some = __ballot(mine.hi > mine.lo);
      const int from = mine.hi > mine.lo ? tid : some ? __ffsll((unsigned long long)some) - 1 : tid;
      slo[tid] = __shfl(mine.lo, from);
      shi[tid] = __shfl(mine.hi, from);
      sbase[tid] = __shfl(mine.base, from);
      rslope[tid] = 0;
      rpos[tid] = 0;
      if constexpr (bias)
        if (g.slope && !more) {
          rslope[tid] = g.slope[mine.head];
          rpos[tid] = g.pos[mine.tok];
        }
    }
    int page = ahead.any() ? page_of(ahead.at) : 0;
    __syncthreads();

    auto load = [&]() {
      if (step == 0) {
        const uint32_t key = min(uint32_t(kb) + uint32_t(li), uint32_t(last));
        in = page >= 0 && page < d.c.n_pages;
        at = ((int64_t(in ? page : 0) * d.c.heads + u.kv) * psize + key % psize) * d.c.dim;
        ahead.advance();
        if (ahead.any()) page = page_of(ahead.at);
      }
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const int w = step * 64 + 4 * G * c;  // first word of the chunk
        if (w < kn) {
          const int i = k0 + w + lg * G;
          if constexpr (Form<F>::y) y[c] = row_group<T, VEC>(g.y + at, i, d.c.dim);
          if constexpr (Form<F>::b0) b0[c] = row_group<T, VEC>(g.b0 + at, i, d.c.dim);
          if constexpr (Form<F>::b1) b1[c] = row_group<T, VEC>(g.b1 + at, i, d.c.dim);
        }
      }
      if (step == steps - 1) {
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int row = 16 * t + 4 * lg + r;
            const uint32_t key = uint32_t(kb) + uint32_t(li);
            const size_t o = size_t(sbase[row] + max(min(key, uint32_t(shi[row] - 1)), uint32_t(slo[row])));
            c0[t][r] = more ? g.out[o] : F == AttnForm::P1 ? g.c1[o] : g.c0[o];
            c1[t][r] = F == AttnForm::BOTH && !more ? g.c1[o] : T(0);
          }
      }
    };
    auto multiply = [&]() {
      if (step == 0) {
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int q = 0; q < NQ; q++) acc[t][q] = v4i_t{0, 0, 0, 0};
      }
      const uint4 *x = xs + step * (NT * NQ * 64) + lane;
#pragma unroll
      for (int e = 0; e < NT; e++) {
        v4i_t bp[NQ];  // the step's planes of the keys
#pragma unroll
        for (int c = 0; c < 4; c++) {  // one dword of every plane from a group of four words
          uint32_t o[NQ];
          const int c0 = c * PAIR, c1 = c0 + PAIR - 1;
          group_planes<T>(right_digits<F, T>(e, y[c0], b0[c0], b1[c0]), right_digits<F, T>(e, y[c1], b0[c1], b1[c1]), o);
#pragma unroll
          for (int q = 0; q < NQ; q++) bp[q][c] = int(o[q]);
        }
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int p = 0; p < NQ; p++) {
            const v4i_t a = v4<T>(x[(t * steps * NT + e) * NQ * 64 + p * 64]);
#pragma unroll
            for (int q = 0; q + p < NQ; q++)
              acc[t][p + q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, bp[q], acc[t][p + q], 0, 0, 0);
          }
      }
      if (step + 1 < steps) return;
      const uint32_t key = uint32_t(kb) + uint32_t(li);
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {  // accumulator register r of lane (li, lg): row 4 lg + r, key li
          const int row = 16 * t + 4 * lg + r;
          if (key < uint32_t(rlo[row]) || key >= uint32_t(rhi[row])) continue;
          T v = (in ? digit_fold<T>(acc[t], r) : T(0)) + c0[t][r];
          if constexpr (F == AttnForm::BOTH) v += c1[t][r];
          if constexpr (bias) v += rslope[row] * T(int64_t(key) - rpos[row]);
          g.out[size_t(rbase[row] + key)] = v;
        }
    };
    kb = ahead.at;
    step = 0;
    if (kb < khi) load();
    put(tid, first);
    for (int e = tid + 64 * kScoreWaves; e < 16 * RT * steps * 16; e += 64 * kScoreWaves) {
      Query q;
      get(e, q);
      put(e, q);
    }
    __syncthreads();
    while (kb < khi) {
      multiply();
      if (++step == steps) step = 0, kb = ahead.at;
      if (kb < khi) load();
    }
  }
}

// ---------------------------------------------------------------------------
// Weighted sums.  A wave takes 64 bytes of keys at a time (16 or 8): their weights as
// the 16 rows' operand, and 256 bytes of columns of the values' rows, lane (li, lg)
// loading group li of the rows lg G .. + G - 1, so that word q of its groups is the
// operand of column tile q.  A value's digits go to the matrix cores as its word holds
// them, each word's bytes beside one another, and the weights' digits shifted against them
// (digit p - s of a weight meets digit s of a value): 16 or 64 MFMAs where planes would
// take 10 or 36, but planes would have to gather a column's bytes from four keys' rows,
// and the MFMAs do not bound it.  The waves of a workgroup and the launch's splits share
// the keys out; their sums meet in LDS and in integer additions to the output, whose order
// does not matter.
// One token a sequence is bound by the cache's bytes: 8 sequences of up to 4096 keys, 8
// heads of 128 in Z_2^32: 71 us a call for 296 MB, 4.2 TB/s (Z_2^64: 143 for 592 MB); one
// of 50000 keys, 4 heads: 66 us, 317 MB at 4.8 TB/s.  Prompts are bound by the digits'
// vector instructions, which every tile of rows repeats: 3 of up to 301 tokens, 6 heads of
// 72 in Z_2^64: 38.4 us.
// (Values' planes staged in LDS for eight tiles of rows were slower, for their longer
// start: 86.8 us against 72.8 for 597 tokens and 1061 keys, 16.4 against 7.3 for 26.)
// Eight waves: four take 94.6 us for the 8 sequences, 58.6 for the prompts.
// ---------------------------------------------------------------------------
constexpr int kMixWaves = 8;
template <AttnForm F, typename T, bool VEC>
__global__ __launch_bounds__(64 * kMixWaves) void k_attn_mix(AttnArgs<T> g, Units units) {
  constexpr int G = 16 / int(sizeof(T)), NQ = int(sizeof(T)), NT = Form<F>::terms, CK = 4 * G;
  // chunks whose digit sums stay exact (Z_2^64, 3 terms); Z_2^32 needs them modulo 2^32 only
  constexpr int kFlush = sizeof(T) == 4 ? INT32_MAX : 4096 / CK;
  __shared__ T red[kMixWaves][G * 4][64];
  const AttnDims &d = g.d;
  const int tid = int(threadIdx.x), lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Unit u = unit_of(d, units);
  const uint32_t m = uint32_t(d.heads) / uint32_t(d.c.heads);
  const int t0 = max(d.qstart[u.b], 0), t1 = min(d.qstart[u.b + 1], d.n_tok);
  const uint32_t n_rows = t1 > t0 ? uint32_t(t1 - t0) * m : 0u;
  const int col = u.col * 16 * G + li * G;  // this lane's columns
  const int32_t *table = d.pages + int64_t(u.b) * d.max_pages;
  const uint32_t psize = uint32_t(d.c.page);
  for (int64_t eb = int64_t(u.tile) * 16; eb < n_rows; eb += int64_t(units.tiles) * 16) {
    const uint32_t e0 = uint32_t(eb);
    const TileRow mine = tile_row(d, t0, t1, u.kv, m, e0 + uint32_t(li));
    int klo, khi;
    tile_keys<16>(mine, klo, khi);
    const int lo = mine.lo, hi = mine.hi;
    // where a weight is read for a row or key without one: some weight of a row that has
    // (a place that others read too, not one that all the GPU reads)
    const uint64_t some = __ballot(hi > lo);
    const int from = hi > lo || !some ? lane : __ffsll((unsigned long long)some) - 1;
    const int slo = __shfl(lo, from), shi = __shfl(hi, from);
    const int64_t sbase = __shfl(mine.base, from);
    KeySteps keys(units, u.split, klo, khi, wave, kMixWaves, CK);
    // a chunk's rows and weights, and the page numbers of the next one
    uint4 y[G], b0[G], b1[G];
    T xw[G], a0w[G], a1w[G];
    uint32_t used = 0;  // bit i: key i of the chunk counts for this lane's row
    int page[G];
    auto pages = [&]() {
#pragma unroll
      for (int i = 0; i < G; i++) {
        const uint32_t key = min(uint32_t(keys.at) + uint32_t(lg * G + i), uint32_t(khi - 1));
        page[i] = table[key / psize];
      }
    };
    auto load = [&]() {
      const uint32_t k0 = uint32_t(keys.at) + uint32_t(lg * G);  // this lane's keys k0 .. k0 + G - 1
      used = 0;
#pragma unroll
      for (int i = 0; i < G; i++) {
        const uint32_t key = min(k0 + i, uint32_t(khi - 1));
        const bool in = page[i] >= 0 && page[i] < d.c.n_pages;
        const int64_t at = ((int64_t(in ? page[i] : 0) * d.c.heads + u.kv) * psize + key % psize) * d.c.dim;
        if constexpr (Form<F>::y) y[i] = row_group<T, VEC>(g.y + at, col, d.c.dim);
        if constexpr (Form<F>::b0) b0[i] = row_group<T, VEC>(g.b0 + at, col, d.c.dim);
        if constexpr (Form<F>::b1) b1[i] = row_group<T, VEC>(g.b1 + at, col, d.c.dim);
        // a weight outside the range, or of a row that is not there: no product
        if (in && k0 + i >= uint32_t(lo) && k0 + i < uint32_t(hi)) used |= 1u << i;
      }
#pragma unroll
      for (int i = 0; i < G; i++) {
        const int64_t o = sbase + max(min(k0 + i, uint32_t(shi - 1)), uint32_t(slo));
        xw[i] = g.x[o];
        a0w[i] = Form<F>::a0 ? g.a0[o] : T(0);
        a1w[i] = Form<F>::a1 ? g.a1[o] : T(0);
      }
      keys.advance();
      if (keys.any()) pages();
    };
    v4i_t acc[G][NQ];
    T vs[G][4];
#pragma unroll
    for (int q = 0; q < G; q++)
#pragma unroll
      for (int r = 0; r < 4; r++) vs[q][r] = 0;
    bool more = keys.any();
    if (more) {
      pages();
      load();
    }
    while (more) {
#pragma unroll
      for (int q = 0; q < G; q++)
#pragma unroll
        for (int s = 0; s < NQ; s++) acc[q][s] = v4i_t{0, 0, 0, 0};
      for (int it = 0; it < kFlush && more; it++) {
        uint4 x, a0, a1;
#pragma unroll
        for (int i = 0; i < G; i++) {
          const bool use = used >> i & 1u;
          xw[i] = use ? xw[i] : T(0);
          a0w[i] = use ? a0w[i] : T(0);
          a1w[i] = use ? a1w[i] : T(0);
        }
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
        more = keys.any();
        if (more) load();
      }
#pragma unroll
      for (int q = 0; q < G; q++)
#pragma unroll
        for (int r = 0; r < 4; r++) vs[q][r] += digit_fold<T>(acc[q], r);
    }
    __syncthreads();  // the last tile's sums are read
#pragma unroll
    for (int q = 0; q < G; q++)
#pragma unroll
      for (int r = 0; r < 4; r++) red[wave][q * 4 + r][lane] = vs[q][r];
    __syncthreads();
    for (int e = tid; e < G * 4 * 64; e += 64 * kMixWaves) {
      // words in the order of the output: row, column (G a lane)
      const int row = e / (16 * G), c = e % (16 * G), q = c % G, l = 16 * (row / 4) + c / G, at = q * 4 + row % 4;
      const int oc = u.col * 16 * G + c;
      const uint32_t er = e0 + uint32_t(row);
      if (er >= n_rows || oc >= d.c.dim) continue;
      const uint32_t qt = er / m;
      T v = 0;
#pragma unroll
      for (int k = 0; k < kMixWaves; k++) v += red[k][at][l];
      const size_t o = size_t((int64_t(t0 + int(qt)) * d.heads + u.kv * int64_t(m) + (er - qt * m)) * d.c.dim + oc);
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
// Rows of a sequence and a cache head by the caller's hint; no sequence has more tokens
// than the batch.
int64_t rows_hint(const AttnDims &d) { return int64_t(std::min(d.max_q, d.n_tok)) * (d.heads / d.c.heads); }
// About `want` units of `threads`, at least one tile and one split for each pair and column
// group, and no more threads than a launch may have; none (n = 0) where the pairs alone
// are too many.
Units units_for(const AttnDims &d, int threads, int cols, int rows, int64_t want, int64_t keys_per_split) {
  Units u;
  const int64_t base = int64_t(d.n_seq) * d.c.heads, most = int64_t(kMostThreads / unsigned(threads));
  if (base > most / cols) return u;
  u.cols = cols;
  u.tiles = int(std::max<int64_t>(1, std::min((rows_hint(d) + rows - 1) / rows, most / (base * cols))));
  const int64_t one = base * cols * u.tiles, keys = (int64_t(d.max_keys) + keys_per_split - 1) / keys_per_split;
  u.splits = int(std::max<int64_t>(1, std::min((want + one - 1) / one, std::min(keys, most / one))));
  u.n = int(one * u.splits);
  return u;
}

// LDS of a launch's queries: 1 KB a plane and step
template <AttnForm F, typename T>
constexpr size_t kStepLds = size_t(Form<F>::terms) * sizeof(T) * 1024;
constexpr size_t kScoreLds = 62 * 1024;

template <AttnForm F, typename T, int RT>
hipError_t scores_rows(const Launch &L, const AttnArgs<T> &g, int dims, int64_t want) {
  const Units u = units_for(g.d, 64 * kScoreWaves, 1, 16 * RT, want, 16 * kScoreWaves);
  if (u.n == 0) return hipErrorInvalidValue;
  const bool vec = vec_rows(g, true);
  for (int k0 = 0; k0 < g.d.c.dim; k0 += dims) {
    const int kn = std::min(dims, g.d.c.dim - k0);
    const size_t lds = kStepLds<F, T> * RT * size_t((kn + 63) / 64);
    if (vec)
      hipLaunchKernelGGL((k_attn_scores<F, T, true, RT>), dim3(unsigned(u.n)), dim3(64 * kScoreWaves), lds, L.stream, g, u,
                         k0, kn, k0 > 0);
    else
      hipLaunchKernelGGL((k_attn_scores<F, T, false, RT>), dim3(unsigned(u.n)), dim3(64 * kScoreWaves), lds, L.stream, g, u,
                         k0, kn, k0 > 0);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
// Two tiles of rows to a workgroup, where LDS holds them: the keys' planes are formed once
// for both.  Z_2^32: from about one workgroup a CU on (4 prompts of 256 tokens against 1024
// keys, 8 heads of 64: 46.6 us, one tile 60.5; 4 of 64 tokens: 23.1, one 20.8); Z_2^64,
// where a key's planes cost more: from 64 rows on (4 of 16 tokens, 4 heads a key: 18.1 us,
// one 22.2; 4 of 8 tokens: 17.1, one 13.2).
template <typename T>
bool two_tiles(const AttnDims &d, int num_cu) {
  const int64_t rows = rows_hint(d);
  if (sizeof(T) == 8) return rows >= 64;
  return int64_t(d.n_seq) * d.c.heads * ((rows + 31) / 32) >= num_cu;
}
template <AttnForm F, typename T>
hipError_t scores_at(const Launch &L, const AttnArgs<T> &g) {
  const size_t steps = size_t(g.d.c.dim + 63) / 64;
  // two workgroups a CU: one takes 97.5 us for 8 tokens against up to 4096 keys each, 8
  // cache heads of 128, two 79.5, four 78.6 but 26.2 for 21.3 for 4 x 64 against 1024
  const int64_t want = int64_t(L.num_cu) * 2;
  if (steps * kStepLds<F, T> * 2 <= kScoreLds && two_tiles<T>(g.d, L.num_cu))
    return scores_rows<F, T, 2>(L, g, g.d.c.dim, want);
  const int dims = int(std::min(steps, kScoreLds / kStepLds<F, T>)) * 64;
  return scores_rows<F, T, 1>(L, g, dims, want);
}
template <AttnForm F, typename T>
hipError_t mix_at(const Launch &L, const AttnArgs<T> &g) {
  constexpr int G = 16 / int(sizeof(T));
  // One workgroup a CU, which its registers allow: half as many take 42.0 us for 4 tokens
  // against 6000 keys, 4 cache heads of 80 (one a CU 28.6), twice as many 32.1.
  // Keys are split down to one step a wave, but not those of four steps at most, where the
  // second launch costs more (one token, 8 heads of 64 in Z_2^32: 2000 keys 12.4 us, split
  // to four steps 18.8; 300 keys 10.7, split 11.9).
  constexpr int64_t kStepKeys = int64_t(kMixWaves) * 4 * G;
  const int64_t part = g.d.max_keys > 4 * kStepKeys ? kStepKeys : 4 * kStepKeys;
  const Units u = units_for(g.d, 64 * kMixWaves, (g.d.c.dim + 16 * G - 1) / (16 * G), 16, int64_t(L.num_cu), part);
  if (u.n == 0) return hipErrorInvalidValue;
  if (u.splits > 1) {
    const size_t n = size_t(g.d.n_tok) * g.d.heads * g.d.c.dim, want = (n + 255) / 256, cap = size_t(L.num_cu) * 32;
    hipLaunchKernelGGL((k_mix_init<F, T>), dim3(unsigned(want < cap ? want : cap)), dim3(256), 0, L.stream, g, n);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (vec_rows(g, false))
    hipLaunchKernelGGL((k_attn_mix<F, T, true>), dim3(unsigned(u.n)), dim3(64 * kMixWaves), 0, L.stream, g, u);
  else
    hipLaunchKernelGGL((k_attn_mix<F, T, false>), dim3(unsigned(u.n)), dim3(64 * kMixWaves), 0, L.stream, g, u);
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
