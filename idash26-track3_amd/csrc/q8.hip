// q8.hip -- masked activations times public 8-bit weights, with a scale for each output
// channel and each token.
//
// C[m, n] = tok[m] scale[n] sum_k q[n, k] A[m, k] mod 2^bw.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn.h"
#include "launch_util.h"

namespace mpcx {
namespace {

template <typename T>
__global__ __launch_bounds__(256) void k_q8(Q8Args<T> g) {
  const int n = int(blockIdx.x) * 256 + int(threadIdx.x), m = int(blockIdx.y);
  if (n >= g.N) return;
  const T *a = g.a + size_t(m) * g.lda;
  const int8_t *q = g.q + size_t(n) * g.ldq;
  T v = 0;
  for (int k = 0; k < g.K; k++) v += a[k] * T(int64_t(q[k]));
  if (g.scale) v *= T(int64_t(g.scale[n]));
  if (g.tok) v *= T(int64_t(g.tok[m]));
  g.c[size_t(m) * g.ldc + n] = v;
}

}  // namespace

template <typename T>
hipError_t launch_gemm_q8(const Launch &L, const Q8Args<T> &g) {
  if (g.K > kQ8MaxK) return hipErrorInvalidValue;
  // a launch has fewer than 2^32 threads along a dimension and 2^16 workgroups along y
  for (int m = 0; m < g.M; m += 1 << 15)
    for (int64_t n = 0; n < g.N; n += 1 << 30) {
      Q8Args<T> p = g;
      p.M = std::min(g.M - m, 1 << 15);
      p.N = int(std::min<int64_t>(g.N - n, 1 << 30));
      p.a += size_t(m) * g.lda;
      p.q += size_t(n) * g.ldq;
      if (p.scale) p.scale += n;
      if (p.tok) p.tok += m;
      p.c += size_t(m) * g.ldc + size_t(n);
      hipLaunchKernelGGL((k_q8<T>), dim3(unsigned((p.N + 255) / 256), unsigned(p.M)), dim3(256), 0, L.stream, p);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  return hipSuccess;
}
template hipError_t launch_gemm_q8<uint32_t>(const Launch &, const Q8Args<uint32_t> &);
template hipError_t launch_gemm_q8<uint64_t>(const Launch &, const Q8Args<uint64_t> &);

}  // namespace mpcx
