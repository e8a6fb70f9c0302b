// q4.hip -- masked activations times public 4-bit weights with group scales.
#include <hip/hip_runtime.h>

#include "attn.h"
#include "launch_util.h"

namespace mpcx {

size_t q4_work_bytes(int, int, int) { return 0; }

// One output per thread: the group's sum of weight times word, then its scale.
template <typename T>
__global__ __launch_bounds__(256) void k_q4(Q4Args<T> g) {
  const int n = int(blockIdx.x) * 256 + int(threadIdx.x);
  if (n >= g.N) return;
  const uint8_t *q = g.q + size_t(n) * ((size_t(g.K) + 31) / 32 * 16);
  for (int m = int(blockIdx.y); m < g.M; m += int(gridDim.y)) {
    const T *a = g.a + size_t(m) * g.lda;
    T out = 0;
    for (int k0 = 0, gi = 0; k0 < g.K; k0 += g.group, gi++) {
      const int k1 = g.K - k0 < g.group ? g.K : k0 + g.group;
      T v = 0;
      for (int k = k0; k < k1; k++) {
        const int w = int((q[k >> 1] >> (4 * (k & 1))) & 15u);
        v += T(int64_t((w ^ 8) - 8)) * a[k];
      }
      out += T(int64_t(g.scale[size_t(gi) * g.N + n])) * v;
    }
    g.c[size_t(m) * g.ldc + n] = out;
  }
}

template <typename T>
hipError_t launch_gemm_q4(const Launch &L, const Q4Args<T> &g) {
  const unsigned gy = unsigned(g.M < 65535 ? g.M : 65535);
  hipLaunchKernelGGL(k_q4<T>, dim3(unsigned((size_t(g.N) + 255) / 256), gy), dim3(256), 0, L.stream, g);
  return hipGetLastError();
}
template hipError_t launch_gemm_q4<uint32_t>(const Launch &, const Q4Args<uint32_t> &);
template hipError_t launch_gemm_q4<uint64_t>(const Launch &, const Q4Args<uint64_t> &);

}  // namespace mpcx
