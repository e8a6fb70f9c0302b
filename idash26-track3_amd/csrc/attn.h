// attn.h -- host-side launchers of the transformer operators: products with
// public 4-bit weights (q4.hip), the paged cache and the attention products
// that read it (attn.hip).
#pragma once
#include "kernels.h"
#include "q4_layout.h"

namespace mpcx {

// HIP's limit on the threads of a launch along one dimension
constexpr size_t kMostThreads = UINT32_MAX;

// ---------------- products with 4-bit weights ----------------
// C[m, n] = sum_g scale[g, n] sum_{k in group g} q[n, k] A[m, k] mod 2^bw.
// q: N rows of q4_row_bytes(K) bytes, weight k of a row in the low (k even) or
// high half of byte k / 2, two's complement; scale: ceil(K / group) x N.
constexpr int kQ4MaxK = 1 << 24;  // a tile's weights lie within 32 bits
template <typename T>
struct Q4Args {
  int M = 0, K = 0, N = 0, group = 0;
  const T *a = nullptr;
  size_t lda = 0;
  const uint8_t *q = nullptr;
  const int32_t *scale = nullptr;
  int lds = 0;  // words between the scales' rows (N, or more for some columns of a product)
  T *c = nullptr;
  size_t ldc = 0;
  void *work = nullptr;  // q4_work_bytes
};
size_t q4_work_bytes(int bw, int M, int K);
template <typename T>
hipError_t launch_gemm_q4(const Launch &L, const Q4Args<T> &g);

// ---------------- paged cache ----------------
// A plane of the cache is n_pages x heads x page x dim ring words: a head's rows
// of a page are contiguous.
struct CacheDims {
  int heads = 0, dim = 0, page = 0;
  int64_t n_pages = 0;
};
constexpr int kMaxPlanes = 8;
template <typename T>
struct AppendArgs {
  CacheDims c;
  size_t n_tok = 0;
  const int64_t *slot = nullptr;
  const int32_t *pos = nullptr;
  // rotation: dims [0, 2 half) turned by the tables' row pos[t], in pairs
  // (2i, 2i + 1) or (i, i + half); the other dims shifted left
  int half = 0, n_pos = 0, shift = 0;
  bool pairs = false;
  const T *cos = nullptr, *sin = nullptr;
  int n_planes = 0;
  const T *rows[kMaxPlanes] = {};
  size_t ld[kMaxPlanes] = {};
  T *pool[kMaxPlanes] = {};
  bool rotate[kMaxPlanes] = {};
};
template <typename T>
hipError_t launch_cache_append(const Launch &L, const AppendArgs<T> &g);

// ---------------- attention products ----------------
struct AttnDims {
  CacheDims c;
  int heads = 0, n_tok = 0, n_seq = 0, max_pages = 0, max_q = 1, max_keys = 1;
  int64_t n_scores = 0;
  const int32_t *pages = nullptr, *qstart = nullptr, *lo = nullptr, *hi = nullptr;
  const int64_t *off = nullptr;
};
// What a launch computes, per output word with left operand x (masked) and
// right operand y (a masked cache plane):
//   BOTH  (x - a0)(y - b0) + c0  +  c1 - x b1 - a1 y   (the revealed product)
//   P0    (x - a0)(y - b0) + c0                        (party 0's message)
//   P1    c1 - x b1 - a1 y                             (party 1's message)
//   DEAL  c0 + x b1 + a1 b0: with x the left mask and c0 the output mask, the
//         product term that the parties share (x (b0 + b1) + c0 - a0 b0)
enum class AttnForm { BOTH, P0, P1, DEAL };
template <typename T>
struct AttnArgs {
  AttnDims d;
  const T *x = nullptr, *a0 = nullptr, *a1 = nullptr;
  const T *y = nullptr, *b0 = nullptr, *b1 = nullptr;
  const T *c0 = nullptr, *c1 = nullptr;
  const T *slope = nullptr;  // scores: + slope[head] (key - pos[token]), forms BOTH and P0
  const int32_t *pos = nullptr;
  T *out = nullptr;
};
template <typename T>
hipError_t launch_attn_scores(const Launch &L, AttnForm form, const AttnArgs<T> &g);
template <typename T>
hipError_t launch_attn_mix(const Launch &L, AttnForm form, const AttnArgs<T> &g);

}  // namespace mpcx
