/* Every value of C that the rows of skl_gemm_mxf4.hip's tiles read and write, walked through on the host: for each number of columns of a wave's
 * part, each number of its rows that exist, each lane and pass. Prints "rows ok" or the first access to a row that is not there. */
#include <cstdio>
#include <vector>

#include "../../skl_amd/csrc/skl_mx_rows.hpp"

template <int TN, int TM>
static bool walk(size_t rsc, size_t csc) {
  using Rows = MxRows<TN>;
  for (unsigned rows = 1; rows <= 32u * TM; ++rows) {
    const size_t last = (rows - 1) * rsc + (32 * TN - 1) * csc;
    std::vector<float> c(last + 1);
    std::vector<int> written(last + 1);
    const auto holds = [&](const float *p, size_t n) {  // n values `csc` apart, all of them values of rows that exist
      for (size_t e = 0; e < n; ++e) {
        const ptrdiff_t at = p - c.data() + (ptrdiff_t)(e * csc);
        if (at < 0 || (size_t)at > last) return false;
      }
      return true;
    };
    for (unsigned lane = 0; lane < 64; ++lane) {
      const Rows mine(c.data(), rsc, csc, lane);
      for (int i = 0; i < TM; ++i)
        for (int n = 0; n < Rows::kPasses; ++n) {
          const unsigned r = 32u * i + (unsigned)n * Rows::kRowsAt;
          if (!holds(mine.readable(r, rows), 4)) {
            std::printf("TN %d: %u rows, lane %u, pass at row %u reads behind C\n", TN, rows, lane, r);
            return false;
          }
          if (!mine.exists(r, rows)) continue;
          if (!holds(mine.row(r), 4) || mine.readable(r, rows) != mine.row(r)) {
            std::printf("TN %d: %u rows, lane %u, pass at row %u writes elsewhere\n", TN, rows, lane, r);
            return false;
          }
          for (size_t e = 0; e < 4; ++e) ++written[(size_t)(mine.row(r) - c.data()) + e * csc];
        }
    }
    for (unsigned i = 0; i < rows; ++i)
      for (unsigned j = 0; j < 32u * TN; ++j)
        if (written[i * rsc + j * csc] != 1) {
          std::printf("TN %d: %u rows, value (%u, %u) written %d times\n", TN, rows, i, j, written[i * rsc + j * csc]);
          return false;
        }
  }
  return true;
}

int main() {
  bool ok = true;
  ok = walk<1, 1>(32, 1) && walk<1, 1>(37, 1) && walk<1, 1>(4096, 1) && walk<1, 1>(67, 2) && ok;
  ok = walk<2, 2>(64, 1) && walk<2, 2>(71, 1) && walk<2, 2>(131, 2) && ok;
  ok = walk<4, 4>(128, 1) && walk<4, 4>(131, 1) && walk<4, 4>(257, 2) && ok;
  if (ok) std::printf("rows ok\n");
  return ok ? 0 : 1;
}
