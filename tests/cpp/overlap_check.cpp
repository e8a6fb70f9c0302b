// Checks csrc/overlap.h against a map of bytes: blocks and rows of every small size
// and distance.
#include <cstdio>
#include <initializer_list>
#include <vector>

#include "overlap.h"

using namespace mpcx;

static const size_t kBase = 4096, kLen = 256;

static void *at(size_t i) { return reinterpret_cast<void *>(kBase + i); }
static void mark(std::vector<char> &m, size_t p, size_t rows, size_t pitch, size_t width) {
  for (size_t r = 0; r < rows; r++)
    for (size_t k = 0; k < width; k++) m[p + r * pitch + k] = 1;
}
static bool meet(const std::vector<char> &a, const std::vector<char> &b) {
  for (size_t i = 0; i < a.size(); i++)
    if (a[i] && b[i]) return true;
  return false;
}

int main() {
  long n = 0, bad = 0;
  struct R {
    size_t rows, pitch, width;
  };
  std::vector<R> kinds;
  for (size_t rows : {0, 1, 2, 3, 5})
    for (size_t pitch : {1, 4, 7, 12})
      for (size_t width : {0, 1, 3, 4, 7, 12})
        if (width <= pitch) kinds.push_back({rows, pitch, width});
  for (const R &a : kinds)
    for (const R &b : kinds)
      for (size_t q = 0; q <= 120; q++, n++) {
        std::vector<char> x(kLen), y(kLen);
        mark(x, 60, a.rows, a.pitch, a.width);
        mark(y, q, b.rows, b.pitch, b.width);
        const ByteRows ra{at(60), a.rows, a.pitch, a.width}, rb{at(q), b.rows, b.pitch, b.width};
        const bool apart = !meet(x, y);
        bool ok = rows_apart(ra, rb) == apart && rows_apart(rb, ra) == apart;
        if (b.rows == 1) ok = ok && rows_apart(ra, at(q), b.width) == apart;
        if (!ok && bad++ < 5)
          std::printf("rows %zu x %zu of %zu at 60, %zu x %zu of %zu at %zu\n", a.rows, a.width, a.pitch, b.rows, b.width,
                      b.pitch, q);
      }
  std::printf("%ld pairs, %ld wrong\n", n, bad);
  return bad != 0;
}
