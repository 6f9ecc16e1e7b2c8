// The loads of the row kernels on rows that start anywhere, walked through on the
// CPU: for every width, row stride, row count and start within a 16-byte granule
// in range, each value that a row's threads read is one of the matrix's K columns,
// and every column of the row is read. Prints the number of layouts, exits 1 on
// the first violation.
#include <cstdio>
#include <vector>

#include "../../tt-flow_b200/csrc/int8_rows_span.h"

using namespace tfb200;

int main() {
  long layouts = 0;
  for (int K = 1; K <= 60; ++K)
    for (int ld = K; ld <= K + 17; ++ld)
      for (int M = 1; M <= 4; ++M)
        for (int start = 0; start < 8; ++start, ++layouts)
          for (int row = 0; row < M; ++row) {
            const RowSpan s = row_span(row, M, K, ld);
            const int phase = (start + row * ld) % 8;
            std::vector<int> seen(K, 0);
            // A thread takes the granules from k - phase and k - phase + 8 for its values k .. k + 7; with the sum
            // formed on granules there is one thread more.
            for (int k = 0; k < K + 8; k += 8)
              for (int half = 0; half < 2; ++half) {
                const int k0 = k - phase + 8 * half;
                if (k0 >= K) continue;
                for (int j = 0; j < 8; ++j) {
                  const int c = k0 + j;
                  if (!whole_granule(s, k0) && (c < 0 || c >= K)) continue;
                  const long at = s.row + c;
                  if (at < 0 || at >= static_cast<long>(M - 1) * ld + K || at % ld >= K) {
                    std::printf("K=%d ld=%d M=%d start=%d row=%d: value %ld is not the matrix's\n", K, ld, M, start,
                                row, at);
                    return 1;
                  }
                  if (c >= 0 && c < K) seen[c] = 1;
                }
              }
            for (int c = 0; c < K; ++c)
              if (!seen[c]) {
                std::printf("K=%d ld=%d M=%d start=%d row=%d: column %d is not read\n", K, ld, M, start, row, c);
                return 1;
              }
          }
  std::printf("OK %ld layouts\n", layouts);
  return 0;
}
