// norm.hip -- the two gates of a root-mean-square norm over masked rows: the residual's
// addition with each row's sum of squares, and each row times its factor.
//
// Beaver gates on public masked values (x + its mask) and shares of the masks.  A square
// needs no second operand's mask: sum (h - r)^2 = sum h^2 - 2 sum h r + sum r^2, so with
// shares a0 + a1 = r the parties' messages are linear in them,
//   p0 = sum h (h - 2 a0) + c0,   p1 = c1 - 2 sum h a1,   c0 + c1 = mask + sum r^2,
// and together sum h (h - 2 (a0 + a1)) + c0 + c1: one multiplication an element.  The
// rows' mask is shared once, by the sums' key; the product with the factors uses the same
// shares.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn.h"
#include "launch_util.h"

namespace mpcx {
namespace {

// 16 bytes of words; rows start at any word, so the loads are not assumed aligned to more.
template <typename T>
struct Words {
  static constexpr int N = 16 / int(sizeof(T));
  T w[N];
  __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(w, p, 16); }
  __device__ __forceinline__ void store(T *p) const { __builtin_memcpy(p, w, 16); }
};

// What a row's sum starts from: the shares of its term that the form adds.
template <NormForm F, typename T>
__device__ __forceinline__ T norm_term(const NormSumsArgs<T> &g, size_t t) {
  T c = 0;
  if constexpr (F != NormForm::P1) c += g.c0[t];
  if constexpr (F == NormForm::BOTH || F == NormForm::P1) c += g.c1[t];
  return c;
}
template <NormForm F, typename T>
__global__ __launch_bounds__(256) void k_norm_terms(NormSumsArgs<T> g) {
  const size_t t = size_t(blockIdx.x) * 256 + threadIdx.x;
  if (t < g.rows) g.s[t] = norm_term<F>(g, t);
}

// ---------------------------------------------------------------------------
// W waves a row (W a power of two; a workgroup is 4 waves or W).  The bytes are all there is
// to it: four words in (three without a residual) and one out (none) for one multiplication.
// 6000 x 4096 in Z_2^32 89 us, 5.5 TB/s (a word a lane instead of 16 bytes: 114); one row of
// 4096 2.8 (by one wave 4.9).  Long rows, where they are few: PARTS a row, of `len` words
// (whole turns of the waves), added up in s, which k_norm_terms has begun; sums modulo 2^bw
// do not depend on their order.
// ---------------------------------------------------------------------------
template <NormForm F, typename T, int W, bool RES, bool PARTS>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void k_norm_sums(NormSumsArgs<T> g, uint32_t parts, size_t len) {
  constexpr int GROUP = W > 4 ? W : 4, ROWS = GROUP / W, N = Words<T>::N;
  __shared__ T part[GROUP];
  const int wave = int(threadIdx.x) >> 6, at = int(threadIdx.x) % (64 * W);
  const size_t units = PARTS ? g.rows * parts : g.rows;
  for (size_t t0 = size_t(blockIdx.x) * ROWS; t0 < units; t0 += size_t(gridDim.x) * ROWS) {
    const size_t t = PARTS ? t0 / parts : t0 + wave / W, start = PARTS ? t0 % parts * len : 0;
    const size_t end = PARTS ? min(start + len, g.dim) : g.dim;
    T sum = 0;
    if (t < g.rows) {
      const T *x = g.x + t * g.ldx, *d = RES ? g.d + t * g.ldd : nullptr;
      const T *a0 = g.a0 + t * g.dim, *a1 = g.a1 + t * g.dim;
      T *h = RES ? g.h + t * g.ldh : nullptr, *copy = F == NormForm::DEAL ? g.copy + t * g.dim : nullptr;
      auto word = [&](T v, T b0, T b1) __attribute__((always_inline)) {
        if constexpr (F == NormForm::BOTH) return v * (v - T(2) * (b0 + b1));
        if constexpr (F == NormForm::P0) return v * (v - T(2) * b0);
        if constexpr (F == NormForm::P1) return T(0) - T(2) * v * b1;
        return v * v;
      };
      constexpr bool A0 = F == NormForm::BOTH || F == NormForm::P0, A1 = F == NormForm::BOTH || F == NormForm::P1;
      size_t j = start + size_t(at) * N;
#pragma unroll 2
      for (; j + N <= end; j += 64 * W * N) {
        Words<T> v, r, b0, b1;
        v.load(x + j);
        if constexpr (RES) r.load(d + j);
        if constexpr (A0) b0.load(a0 + j);
        if constexpr (A1) b1.load(a1 + j);
#pragma unroll
        for (int i = 0; i < N; i++) {
          if constexpr (RES) v.w[i] += r.w[i];
          sum += word(v.w[i], A0 ? b0.w[i] : T(0), A1 ? b1.w[i] : T(0));
        }
        if constexpr (RES) v.store(h + j);
        if constexpr (F == NormForm::DEAL) v.store(copy + j);
      }
      for (; j < end; j++) {  // one lane's, fewer than N
        T v = x[j];
        if constexpr (RES) v += d[j];
        sum += word(v, A0 ? a0[j] : T(0), A1 ? a1[j] : T(0));
        if constexpr (RES) h[j] = v;
        if constexpr (F == NormForm::DEAL) copy[j] = v;
      }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if constexpr (W > 1) {
      if (threadIdx.x % 64 == 0) part[wave] = sum;
      __syncthreads();
      sum = 0;
      if (at == 0)
#pragma unroll
        for (int w = 0; w < W; w++) sum += part[wave + w];
      __syncthreads();
    }
    if (at == 0 && t < g.rows) {
      if constexpr (PARTS) {
        using A = std::conditional_t<sizeof(T) == 4, unsigned, unsigned long long>;
        atomicAdd(reinterpret_cast<A *>(g.s + t), A(sum));
      } else {
        g.s[t] = sum + norm_term<F>(g, t);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// A workgroup takes 256 groups of 16 bytes of a row at a time.  Bound by its bytes, too:
// five words in and one out.  6000 x 4096 in Z_2^32 107 us, 5.5 TB/s (a word a lane, its row
// by a division: 116); one row of 4096 2.4.
// ---------------------------------------------------------------------------
template <NormForm F, typename T, bool GAIN>
__global__ __launch_bounds__(256) void k_norm_scale(NormScaleArgs<T> g, uint32_t chunks) {
  constexpr int N = Words<T>::N;
  constexpr bool P0 = F != NormForm::P1, P1 = F == NormForm::BOTH || F == NormForm::P1, DEAL = F == NormForm::DEAL;
  const size_t units = g.rows * chunks;
  for (size_t u = blockIdx.x; u < units; u += gridDim.x) {
    const size_t t = u / chunks, j = (u % chunks * 256 + threadIdx.x) * N, i = t * g.dim + j;
    if (j >= g.dim) continue;
    const T v = g.v[t], b0 = P0 ? g.b0[t] : T(0), b1 = P1 ? g.b1[t] : T(0);
    const T *h = DEAL ? nullptr : g.h + t * g.ldh;
    T *y = g.y + t * g.ldy;
    auto word = [&](T x, T a0, T a1, T c0, T c1, T gain) __attribute__((always_inline)) {
      T z = 0;
      if constexpr (DEAL) {
        z = (a0 + a1) * v - a0 * b0;
      } else {
        if constexpr (P0) z += (x - a0) * (v - b0);
        if constexpr (P1) z -= x * b1 + a1 * v;
      }
      if constexpr (GAIN) z *= gain;
      return z + c0 + c1;
    };
    if (j + N <= g.dim) {
      Words<T> x = {}, a0 = {}, a1 = {}, c0 = {}, c1 = {}, gain = {};
      if constexpr (!DEAL) x.load(h + j);
      if constexpr (P0) a0.load(g.a0 + i), c0.load(g.c0 + i);
      if constexpr (P1 || DEAL) a1.load(g.a1 + i);
      if constexpr (P1) c1.load(g.c1 + i);
      if constexpr (GAIN) gain.load(g.gain + j);
#pragma unroll
      for (int k = 0; k < N; k++) x.w[k] = word(x.w[k], a0.w[k], a1.w[k], c0.w[k], c1.w[k], gain.w[k]);
      x.store(y + j);
    } else {
      for (size_t k = 0; j + k < g.dim; k++)
        y[j + k] = word(DEAL ? T(0) : h[j + k], P0 ? g.a0[i + k] : T(0), P1 || DEAL ? g.a1[i + k] : T(0),
                        P0 ? g.c0[i + k] : T(0), P1 ? g.c1[i + k] : T(0), GAIN ? g.gain[j + k] : T(0));
    }
  }
}

}  // namespace

namespace {
template <NormForm F, typename T, bool RES>
hipError_t sums_form(const Launch &L, const NormSumsArgs<T> &g) {
  auto waves = [&](auto w) {
    constexpr int W = decltype(w)::value, ROWS = W > 4 ? 1 : 4 / W;
    const size_t want = (g.rows + ROWS - 1) / ROWS, cap = size_t(L.num_cu) * 16;
    hipLaunchKernelGGL((k_norm_sums<F, T, W, RES, false>), dim3(unsigned(std::min(want, cap))), dim3(64 * std::max(W, 4)), 0,
                       L.stream, g, 1u, g.dim);
    return hipGetLastError();
  };
  const size_t turns = (g.dim * sizeof(T) + 1023) / 1024;  // of a wave, to pass a row
  // Long rows in parts, a workgroup each, where the rows leave CUs idle (us, whole and in parts,
  // Z_2^32): 1 row of 16384 4.6 and 4.8, of 32768 7.3 and 4.8, of 262144 55 and 5.3; 16 rows of 32768 8.6 and
  // 6.2; 64 rows 10.8 and 10.5; 128 rows 13.8 and 16.2, of 65536 35 and 30; 256 rows 66 and 69.
  const size_t rounds = (turns + 15) / 16, cus = size_t(L.num_cu);  // of 16 waves, to pass a row
  if (rounds >= 8 && g.rows <= cus * std::min<size_t>(rounds, 16) / 32) {
    const size_t most = std::min(rounds, (cus + g.rows - 1) / g.rows), len = (rounds + most - 1) / most * (16384 / sizeof(T));
    const size_t parts = (g.dim + len - 1) / len;
    hipLaunchKernelGGL((k_norm_terms<F, T>), dim3(unsigned((g.rows + 255) / 256)), dim3(256), 0, L.stream, g);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_norm_sums<F, T, 16, RES, true>), dim3(unsigned(g.rows * parts)), dim3(1024), 0, L.stream, g,
                       uint32_t(parts), len);
    return hipGetLastError();
  }
  // By 16, 4 and 1 waves (us, Z_2^32): 1 x 4096 2.8, 3.0, 4.9; 2000 x 4096 27, 27, 28; 8000 x
  // 4096 120, 125, 132; 700 x 2048 7.6, 6.7, 6.6; 8000 x 1024 32, 28, 27; 8000 x 128 23, 9.2, 5.4.
  if (turns > 8) return waves(std::integral_constant<int, 16>{});
  if (turns > 2) return waves(std::integral_constant<int, 4>{});
  return waves(std::integral_constant<int, 1>{});
}
}  // namespace

template <typename T>
hipError_t launch_norm_sums(const Launch &L, NormForm form, const NormSumsArgs<T> &g) {
  auto with = [&](auto res) {
    constexpr bool RES = decltype(res)::value;
    switch (form) {
      case NormForm::BOTH: return sums_form<NormForm::BOTH, T, RES>(L, g);
      case NormForm::P0: return sums_form<NormForm::P0, T, RES>(L, g);
      case NormForm::P1: return sums_form<NormForm::P1, T, RES>(L, g);
      default: return sums_form<NormForm::DEAL, T, RES>(L, g);
    }
  };
  return g.d ? with(std::true_type{}) : with(std::false_type{});
}
template <typename T>
hipError_t launch_norm_scale(const Launch &L, NormForm form, const NormScaleArgs<T> &g) {
  const uint32_t chunks = uint32_t((g.dim * sizeof(T) + 4095) / 4096);
  const dim3 grid(unsigned(std::min<size_t>(g.rows * chunks, size_t(L.num_cu) * 64)));
  auto with = [&](auto gain) {
    constexpr bool GAIN = decltype(gain)::value;
    auto launch = [&](auto f) {
      hipLaunchKernelGGL((k_norm_scale<decltype(f)::value, T, GAIN>), grid, dim3(256), 0, L.stream, g, chunks);
      return hipGetLastError();
    };
    switch (form) {
      case NormForm::BOTH: return launch(std::integral_constant<NormForm, NormForm::BOTH>{});
      case NormForm::P0: return launch(std::integral_constant<NormForm, NormForm::P0>{});
      case NormForm::P1: return launch(std::integral_constant<NormForm, NormForm::P1>{});
      default: return launch(std::integral_constant<NormForm, NormForm::DEAL>{});
    }
  };
  return g.gain ? with(std::true_type{}) : with(std::false_type{});
}
template hipError_t launch_norm_sums<uint32_t>(const Launch &, NormForm, const NormSumsArgs<uint32_t> &);
template hipError_t launch_norm_sums<uint64_t>(const Launch &, NormForm, const NormSumsArgs<uint64_t> &);
template hipError_t launch_norm_scale<uint32_t>(const Launch &, NormForm, const NormScaleArgs<uint32_t> &);
template hipError_t launch_norm_scale<uint64_t>(const Launch &, NormForm, const NormScaleArgs<uint64_t> &);

}  // namespace mpcx
