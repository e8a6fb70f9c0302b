// Checks the places that the 4-bit weight products read (csrc/q4_layout.h): every
// lane group's bytes of every chunk lie in the row and where its weights are.
#include <cstdio>
#include <initializer_list>

#include "q4_layout.h"

int main() {
  using namespace mpcx;
  long bad = 0, n = 0;
  for (int S : {32, 64, 128})
    for (int K = 1; K <= 1100; K++) {
      const uint32_t row = uint32_t(q4_row_bytes(K));
      for (int c = 0; c * S < K; c++)
        for (int lg = 0; lg < 4; lg++, n++) {
          const uint32_t at = q4_place(row, S, c, lg);
          const uint32_t first = uint32_t(c * S + lg * (S / 4)) / 2;  // byte of the lane group's first weight
          bool ok = size_t(at) + size_t(S / 8) <= row && at % uint32_t(S / 8) == 0;
          if (c * S + lg * (S / 4) < K) ok = ok && at == first;
          if (!ok && bad++ < 5)
            std::printf("S %d K %d chunk %d lane group %d: bytes %u..%u of a row of %u\n", S, K, c, lg, at,
                        at + uint32_t(S / 8) - 1, row);
        }
    }
  std::printf("%ld places, %ld outside\n", n, bad);
  return bad != 0;
}
