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

#include "attn.h"
#include "launch_util.h"

namespace mpcx {
namespace {

// A wave a row.
template <NormForm F, typename T>
__global__ __launch_bounds__(256) void k_norm_sums(NormSumsArgs<T> g) {
  const size_t waves = size_t(gridDim.x) * 4;
  const int lane = int(threadIdx.x) & 63;
  for (size_t t = size_t(blockIdx.x) * 4 + (threadIdx.x >> 6); t < g.rows; t += waves) {
    T sum = 0;
    for (size_t j = lane; j < g.dim; j += 64) {
      T h = g.x[t * g.ldx + j];
      if (g.d) h += g.d[t * g.ldd + j];
      const size_t i = t * g.dim + j;
      if constexpr (F == NormForm::BOTH) sum += h * (h - T(2) * (g.a0[i] + g.a1[i]));
      if constexpr (F == NormForm::P0) sum += h * (h - T(2) * g.a0[i]);
      if constexpr (F == NormForm::P1) sum -= T(2) * h * g.a1[i];
      if constexpr (F == NormForm::DEAL) sum += h * h, g.copy[i] = h;
      if (g.h) g.h[t * g.ldh + j] = h;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) {
      if constexpr (F != NormForm::P1) sum += g.c0[t];
      if constexpr (F == NormForm::BOTH || F == NormForm::P1) sum += g.c1[t];
      g.s[t] = sum;
    }
  }
}

template <NormForm F, typename T>
__global__ __launch_bounds__(256) void k_norm_scale(NormScaleArgs<T> g) {
  const size_t n = g.rows * g.dim;
  for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += size_t(gridDim.x) * 256) {
    const size_t t = i / g.dim, j = i % g.dim;
    const T v = g.v[t];
    T z = 0;
    if constexpr (F != NormForm::DEAL) {
      const T h = g.h[t * g.ldh + j];
      if constexpr (F != NormForm::P1) z += (h - g.a0[i]) * (v - g.b0[t]);
      if constexpr (F != NormForm::P0) z -= h * g.b1[t] + g.a1[i] * v;
    } else {
      z = (g.a0[i] + g.a1[i]) * v - g.a0[i] * g.b0[t];
    }
    if (g.gain) z *= g.gain[j];
    if constexpr (F != NormForm::P1) z += g.c0[i];
    if constexpr (F == NormForm::BOTH || F == NormForm::P1) z += g.c1[i];
    g.y[t * g.ldy + j] = z;
  }
}

}  // namespace

template <typename T>
hipError_t launch_norm_sums(const Launch &L, NormForm form, const NormSumsArgs<T> &g) {
  const dim3 grid(unsigned(std::min<size_t>((g.rows + 3) / 4, size_t(L.num_cu) * 8)));
  switch (form) {
    case NormForm::BOTH: hipLaunchKernelGGL((k_norm_sums<NormForm::BOTH, T>), grid, dim3(256), 0, L.stream, g); break;
    case NormForm::P0: hipLaunchKernelGGL((k_norm_sums<NormForm::P0, T>), grid, dim3(256), 0, L.stream, g); break;
    case NormForm::P1: hipLaunchKernelGGL((k_norm_sums<NormForm::P1, T>), grid, dim3(256), 0, L.stream, g); break;
    case NormForm::DEAL: hipLaunchKernelGGL((k_norm_sums<NormForm::DEAL, T>), grid, dim3(256), 0, L.stream, g); break;
  }
  return hipGetLastError();
}
template <typename T>
hipError_t launch_norm_scale(const Launch &L, NormForm form, const NormScaleArgs<T> &g) {
  const dim3 grid(unsigned(std::min<size_t>((g.rows * g.dim + 255) / 256, size_t(L.num_cu) * 8)));
  switch (form) {
    case NormForm::BOTH: hipLaunchKernelGGL((k_norm_scale<NormForm::BOTH, T>), grid, dim3(256), 0, L.stream, g); break;
    case NormForm::P0: hipLaunchKernelGGL((k_norm_scale<NormForm::P0, T>), grid, dim3(256), 0, L.stream, g); break;
    case NormForm::P1: hipLaunchKernelGGL((k_norm_scale<NormForm::P1, T>), grid, dim3(256), 0, L.stream, g); break;
    case NormForm::DEAL: hipLaunchKernelGGL((k_norm_scale<NormForm::DEAL, T>), grid, dim3(256), 0, L.stream, g); break;
  }
  return hipGetLastError();
}
template hipError_t launch_norm_sums<uint32_t>(const Launch &, NormForm, const NormSumsArgs<uint32_t> &);
template hipError_t launch_norm_sums<uint64_t>(const Launch &, NormForm, const NormSumsArgs<uint64_t> &);
template hipError_t launch_norm_scale<uint32_t>(const Launch &, NormForm, const NormScaleArgs<uint32_t> &);
template hipError_t launch_norm_scale<uint64_t>(const Launch &, NormForm, const NormScaleArgs<uint64_t> &);

}  // namespace mpcx
