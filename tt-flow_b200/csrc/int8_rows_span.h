// Which values of a bf16 matrix the row kernels may read sixteen bytes at a time
// (int8_rows.cu, rows that start anywhere). Plain C++ apart from the qualifiers;
// tests/native/int8_span_check.cpp checks it on the CPU.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define TFB_SPAN_HD __host__ __device__ __forceinline__
#else
#define TFB_SPAN_HD inline
#endif

namespace tfb200 {

// A row of a matrix [M, K] with its rows ld apart, as offsets from the matrix's
// start: its first value, and the values around it that belong to the matrix.
// Only the K columns of a row are the operator's to read: where rows are padded
// these are the row's own, where they follow each other the whole matrix.
struct RowSpan {
  int64_t row, lo, hi;
};
TFB_SPAN_HD RowSpan row_span(int64_t row, int64_t M, int64_t K, int64_t ld) {
  if (ld == K) return {row * ld, 0, M * K};
  return {row * ld, row * ld, row * ld + K};
}

// Whether the eight values from column k of the row (k may be negative) all are
// in its span; if not, those of columns 0 .. K - 1 are read one by one.
TFB_SPAN_HD bool whole_granule(const RowSpan& s, int64_t k) {
  return s.row + k >= s.lo && s.row + k + 8 <= s.hi;
}

}  // namespace tfb200
