// Host-side interfaces of the 8-bit integer path: row quantisation, RMSNorm
// with an int8 result, and the int8 matrix product. Shared by int8_*.cu.
#pragma once

#include "internal.h"

namespace tfb200 {

// What a product's epilogue writes: bf16 or fp32 for the caller, or the fused
// MLP's hidden block (Int8Hidden).
enum Int8Out : int { kInt8OutBf16 = 0, kInt8OutF32 = 1, kInt8OutHidden = 2 };

// Longest inner dimension: |sum_k a b| <= 128 * 128 * K must stay in int32.
constexpr int64_t kInt8MaxK = 131071;

// The hidden block between an MLP's products, which is quantised again per row
// once the whole row is known: 16-bit integers with the largest magnitude of
// each 32 columns of a row beside them, h = value * max / 32767. That is as many
// bytes as bf16 and keeps h to 2^-16 of its neighbourhood: with fp16 (bf16) the
// second quantisation moved about 0.5 % (2 %) of the values by an int8 step, here
// under 0.1 %. It holds the whole range of fp32; a block of 32 with an infinity
// or a NaN has maximum NaN.
constexpr int kHiddenBlock = 32;
struct Int8Hidden {
  int64_t ld = 0, ldm = 0;  // row strides of the values and of the maxima
  size_t max_at = 0, bytes = 0;
};
inline Int8Hidden int8_hidden(int64_t m, int64_t h) {
  Int8Hidden l;
  l.ld = (h + 15) / 16 * 16;
  l.ldm = (h + 127) / 128 * 4;  // four maxima at a time
  l.max_at = (static_cast<size_t>(m) * l.ld * 2 + 255) / 256 * 256;
  l.bytes = l.max_at + static_cast<size_t>(m) * l.ldm * 4;
  return l;
}

// v = a_scale[m] * b_scale[n] * sum_k A[m,k] B[n,k], then + bias[n], GELU and
// + residual[m,n] (each optional). A [M,K] and B [N,K] are int8, row-major.
struct Int8Gemm {
  int64_t M = 0, N = 0, K = 0;
  const int8_t* A = nullptr;
  int64_t lda = 0;
  const int8_t* B = nullptr;
  int64_t ldb = 0;
  const float* a_scale = nullptr;
  const float* b_scale = nullptr;
  const bf16* bias = nullptr;
  int gelu = kGeluNone;
  const bf16* residual = nullptr;
  int64_t ldr = 0;
  void* C = nullptr;
  int64_t ldc = 0;
  int out = kInt8OutBf16;
  float* hidden_max = nullptr;  // kInt8OutHidden: maxima, ldm apart
  int64_t ldm = 0;
  void* ws = nullptr;            // int8_gemm_ws(M, N, K).total bytes, 256-byte aligned, its counters cleared
  // The kernel that precedes this product in the stream writes neither B nor
  // b_scale (it is this library's own staging launch), so their first tiles may
  // be requested before it has completed.
  bool b_stable = false;
  bool a_stable = false;  // nor A (a bare product behind the clear of its counters)
  // Few rows only: the weights [next_n, next_k] of the product that follows on
  // the stream, the first of which are brought into L2 while this one drains.
  const int8_t* next_b = nullptr;
  int64_t next_n = 0, next_k = 0, next_ld = 0;
};

// Device workspace of one product: `clear_bytes` of counters, zero on entry,
// then its partial-sum slots.
struct Int8GemmWs {
  size_t clear_bytes = 0, total = 0;
};
Int8GemmWs int8_gemm_ws(int64_t m, int64_t n, int64_t k, bool hidden = false);
int run_int8_gemm(const Int8Gemm& g, cudaStream_t stream, std::string* err);

// Few rows (int8_stream.cu); operands as run_int8_gemm checks them for TMA.
constexpr int64_t kInt8StreamRows = 128;
Int8GemmWs int8_stream_ws(int64_t m, int64_t n);
int run_int8_stream(const Int8Gemm& g, cudaStream_t stream, std::string* err);
// A handful of rows (int8_gemv.cu); operands as above, no workspace.
constexpr int64_t kInt8GemvRows = 32;
double int8_gemv_us(int64_t m, int64_t n, int64_t k, bool hidden);  // estimate
int run_int8_gemv(const Int8Gemm& g, cudaStream_t stream, std::string* err);
// Tensor map of an int8 matrix in boxes of 128 columns (int8_gemm.cu).
bool int8_map(CUtensorMap* m, const int8_t* base, int64_t rows, int64_t cols, int64_t ld, uint32_t box_rows,
              std::string* err);

// One row at a time: q = rn(t * 127 / amax_k |t|) with t = x (kInt8RowsQuant),
// t = (x + residual) * gamma with scale = amax / (127 rms) (kInt8RowsNorm), or
// t = the fused MLP's hidden block (kInt8RowsHidden).
enum Int8RowsKind : int { kInt8RowsQuant = 0, kInt8RowsNorm = 1, kInt8RowsHidden = 2 };
struct Int8Rows {
  int kind = kInt8RowsQuant;
  int64_t M = 0, K = 0;
  const void* x = nullptr;
  int64_t ldx = 0;
  const bf16* residual = nullptr;  // kInt8RowsNorm, optional
  int64_t ldr = 0;
  const bf16* gamma = nullptr;
  float eps = 0.0f;
  bf16* sum = nullptr;  // bf16(x + residual), with a residual
  int64_t lds = 0;
  int8_t* q = nullptr;
  int64_t ldq = 0;
  float* scale = nullptr;
  const float* hidden_max = nullptr;  // kInt8RowsHidden
  int64_t ldm = 0;
  // Optional: counters of the products that follow, cleared by the same launch
  // (16-byte aligned, a multiple of 16 bytes).
  void* zero = nullptr;
  size_t zero_bytes = 0;
};
// Clears `bytes` (16-byte aligned, a multiple of 16) ahead of a bare product.
int run_int8_clear(void* p, size_t bytes, cudaStream_t stream, std::string* err);
int run_int8_rows(const Int8Rows& r, cudaStream_t stream, std::string* err);

}  // namespace tfb200
