// attn.h -- host-side launchers of the transformer operators: products with
// public 4-bit (q4.hip) and 8-bit weights (q8.hip), the paged cache and the
// attention products that read it (attn.hip), the norm's gates (norm.hip).
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

// ---------------- products with 8-bit weights ----------------
// C[m, n] = tok[m] scale[n] sum_k q[n, k] A[m, k] mod 2^bw; scale, tok may be null (1).
constexpr int kQ8MaxK = 1 << 24;
template <typename T>
struct Q8Args {
  int M = 0, K = 0, N = 0;
  const T *a = nullptr;
  size_t lda = 0;
  const int8_t *q = nullptr;  // rows of K weights, ldq (a multiple of 16) bytes apart
  size_t ldq = 0;
  const int32_t *scale = nullptr, *tok = nullptr;
  T *c = nullptr;
  size_t ldc = 0;
};
template <typename T>
hipError_t launch_gemm_q8(const Launch &L, const Q8Args<T> &g);

// ---------------- the norm's gates ----------------
// The keygens' PRF fields, beside the enum Field's: share 0 of the rows' (the factors') mask, the
// output's mask (+1), share 0 of the term (+2).  With fields of their own a norm's two gates
// may have one gate id.
constexpr uint32_t F_NSUMS = 0x68, F_NSCALE = 0x6C;
// What a launch computes: both parties' messages added up, one party's, or the
// dealer's product term.
enum class NormForm { BOTH, P0, P1, DEAL };
// h = x + d (d may be null: h = x) and s[t] = sum_j h[t, j]^2, as
//   P0    sum h (h - 2 a0) + c0
//   P1    c1 - 2 sum h a1
//   DEAL  sum h^2 + c0, and h to `copy`: with x, d masks and c0 the sums' mask
template <typename T>
struct NormSumsArgs {
  size_t rows = 0, dim = 0;
  const T *x = nullptr, *d = nullptr;
  size_t ldx = 0, ldd = 0;
  const T *a0 = nullptr, *a1 = nullptr, *c0 = nullptr, *c1 = nullptr;
  T *h = nullptr;  // may be null, x or d
  size_t ldh = 0;
  T *copy = nullptr;
  T *s = nullptr;
};
template <typename T>
hipError_t launch_norm_sums(const Launch &L, NormForm form, const NormSumsArgs<T> &g);
// y[t, j] = gain[j] h[t, j] v[t] (gain may be null: 1), as
//   P0    gain (h - a0)(v - b0) + c0
//   P1    c1 - gain (h b1 + a1 v)
//   DEAL  c0 + gain ((a0 + a1) v - a0 b0): with v the factors' mask and c0 the output's
template <typename T>
struct NormScaleArgs {
  size_t rows = 0, dim = 0;
  const T *h = nullptr;
  size_t ldh = 0;
  const T *a0 = nullptr, *a1 = nullptr, *v = nullptr, *b0 = nullptr, *b1 = nullptr;
  const T *c0 = nullptr, *c1 = nullptr, *gain = nullptr;
  T *y = nullptr;  // may be h
  size_t ldy = 0;
};
template <typename T>
hipError_t launch_norm_scale(const Launch &L, NormForm form, const NormScaleArgs<T> &g);

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
