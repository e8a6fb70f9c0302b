// attn.hip -- the paged cache of masked keys and values, and the attention
// products that read it (Beaver gates of both parties).
#include <hip/hip_runtime.h>

#include "attn.h"
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
// word index of row `key` of sequence b's kv head in a cache plane, -1 where the
// page is not in the cache
__device__ __forceinline__ int64_t cache_row(const AttnDims &d, int b, int head, int key) {
  const int page = d.pages[int64_t(b) * d.max_pages + key / d.c.page];
  if (page < 0 || page >= d.c.n_pages) return -1;
  return ((int64_t(page) * d.c.heads + head) * d.c.page + key % d.c.page) * d.c.dim;
}

template <AttnForm F, typename T>
__device__ __forceinline__ T attn_term(const AttnArgs<T> &g, size_t i, int64_t j) {
  const T x = g.x[i];
  if constexpr (F == AttnForm::P0) return (x - g.a0[i]) * (g.y[j] - g.b0[j]);
  if constexpr (F == AttnForm::P1) return T(0) - x * g.b1[j] - g.a1[i] * g.y[j];
  if constexpr (F == AttnForm::DEAL) return x * g.b1[j] + g.a1[i] * g.b0[j];
  return (x - g.a0[i]) * (g.y[j] - g.b0[j]) - x * g.b1[j] - g.a1[i] * g.y[j];
}
template <AttnForm F, typename T>
__device__ __forceinline__ T attn_start(const AttnArgs<T> &g, size_t i) {
  if constexpr (F == AttnForm::P1) return g.c1[i];
  if constexpr (F == AttnForm::BOTH) return g.c0[i] + g.c1[i];
  return g.c0[i];
}

// one workgroup per sequence, token of it and head; one thread per key
template <AttnForm F, typename T>
__global__ __launch_bounds__(256) void k_attn_scores(AttnArgs<T> g) {
  const AttnDims &d = g.d;
  const int b = int(blockIdx.z), h = int(blockIdx.y), group = d.heads / d.c.heads;
  const int t0 = d.qstart[b] < 0 ? 0 : d.qstart[b], t1 = d.qstart[b + 1] < d.n_tok ? d.qstart[b + 1] : d.n_tok;
  for (int t = t0 + int(blockIdx.x); t < t1; t += int(gridDim.x)) {
    const TokenRange r = token_range(d, t);
    for (int key = r.lo + int(threadIdx.x); key < r.hi; key += 256) {
      const int64_t j = cache_row(d, b, h / group, key);
      const size_t i = (size_t(t) * d.heads + h) * d.c.dim, o = size_t(r.off) + size_t(h) * (r.hi - r.lo) + (key - r.lo);
      T v = attn_start<F>(g, o);
      if (j >= 0)
        for (int k = 0; k < d.c.dim; k++) v += attn_term<F>(g, i + k, j + k);
      if constexpr (F == AttnForm::BOTH || F == AttnForm::P0)
        if (g.slope) v += g.slope[h] * T(int64_t(key) - g.pos[t]);
      g.out[o] = v;
    }
  }
}
// one thread per dim
template <AttnForm F, typename T>
__global__ __launch_bounds__(256) void k_attn_mix(AttnArgs<T> g) {
  const AttnDims &d = g.d;
  const int b = int(blockIdx.z), h = int(blockIdx.y), group = d.heads / d.c.heads;
  const int t0 = d.qstart[b] < 0 ? 0 : d.qstart[b], t1 = d.qstart[b + 1] < d.n_tok ? d.qstart[b + 1] : d.n_tok;
  for (int t = t0 + int(blockIdx.x); t < t1; t += int(gridDim.x)) {
    const TokenRange r = token_range(d, t);
    for (int k = int(threadIdx.x); k < d.c.dim; k += 256) {
      const size_t o = (size_t(t) * d.heads + h) * d.c.dim + k;
      T v = attn_start<F>(g, o);
      for (int key = r.lo; key < r.hi; key++) {
        const int64_t j = cache_row(d, b, h / group, key);
        if (j >= 0) v += attn_term<F>(g, size_t(r.off) + size_t(h) * (r.hi - r.lo) + (key - r.lo), j + k);
      }
      g.out[o] = v;
    }
  }
}

#define ATTN_FORMS(KERNEL)                                                                                          \
  switch (form) {                                                                                                   \
    case AttnForm::BOTH: hipLaunchKernelGGL((KERNEL<AttnForm::BOTH, T>), grid, dim3(256), 0, L.stream, g); break;   \
    case AttnForm::P0: hipLaunchKernelGGL((KERNEL<AttnForm::P0, T>), grid, dim3(256), 0, L.stream, g); break;       \
    case AttnForm::P1: hipLaunchKernelGGL((KERNEL<AttnForm::P1, T>), grid, dim3(256), 0, L.stream, g); break;       \
    case AttnForm::DEAL: hipLaunchKernelGGL((KERNEL<AttnForm::DEAL, T>), grid, dim3(256), 0, L.stream, g); break;   \
  }                                                                                                                 \
  return hipGetLastError()

template <typename T>
hipError_t launch_attn_scores(const Launch &L, AttnForm form, const AttnArgs<T> &g) {
  const dim3 grid(unsigned(g.d.max_q), unsigned(g.d.heads), unsigned(g.d.n_seq));
  ATTN_FORMS(k_attn_scores);
}
template <typename T>
hipError_t launch_attn_mix(const Launch &L, AttnForm form, const AttnArgs<T> &g) {
  const dim3 grid(unsigned(g.d.max_q), unsigned(g.d.heads), unsigned(g.d.n_seq));
  ATTN_FORMS(k_attn_mix);
}

#define INST(T)                                                                                       \
  template hipError_t launch_cache_append<T>(const Launch &, const AppendArgs<T> &);                  \
  template hipError_t launch_attn_scores<T>(const Launch &, AttnForm, const AttnArgs<T> &);           \
  template hipError_t launch_attn_mix<T>(const Launch &, AttnForm, const AttnArgs<T> &);
INST(uint32_t)
INST(uint64_t)

}  // namespace mpcx
