// Host-side interfaces of the 8-bit integer path: row quantisation, RMSNorm
// with an int8 result, and the int8 matrix product. Shared by int8_*.cu.
#pragma once

#include "internal.h"

namespace tfb200 {

// What a product's epilogue writes. The fused MLP's hidden block is fp32.
enum Int8Out : int { kInt8OutBf16 = 0, kInt8OutF32 = 1 };

// Longest inner dimension: |sum_k a b| <= 128 * 128 * K must stay in int32.
constexpr int64_t kInt8MaxK = 131071;

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
Int8GemmWs int8_gemm_ws(int64_t m, int64_t n, int64_t k);
int run_int8_gemm(const Int8Gemm& g, cudaStream_t stream, std::string* err);

// Few rows (int8_stream.cu); operands as run_int8_gemm checks them for TMA.
constexpr int64_t kInt8StreamRows = 128;
Int8GemmWs int8_stream_ws(int64_t m, int64_t n);
int run_int8_stream(const Int8Gemm& g, cudaStream_t stream, std::string* err);
// A handful of rows (int8_gemv.cu); operands as above, no workspace.
constexpr int64_t kInt8GemvRows = 32;
double int8_gemv_us(int64_t m, int64_t n, int64_t k);  // estimate
int run_int8_gemv(const Int8Gemm& g, cudaStream_t stream, std::string* err);
// Tensor map of an int8 matrix in boxes of 128 columns (int8_gemm.cu).
bool int8_map(CUtensorMap* m, const int8_t* base, int64_t rows, int64_t cols, int64_t ld, uint32_t box_rows,
              std::string* err);

// One row at a time: q = rn(t * 127 / amax_k |t|) with t = x (kInt8RowsQuant),
// t = (x + residual) * gamma with scale = amax / (127 rms) (kInt8RowsNorm), or
// t = the fp32 rows of the fused MLP's hidden block (kInt8RowsHidden; they start
// on 32-byte boundaries).
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
  // Optional: counters of the products that follow, cleared by the same launch
  // (16-byte aligned, a multiple of 16 bytes).
  void* zero = nullptr;
  size_t zero_bytes = 0;
};
// Clears `bytes` (16-byte aligned, a multiple of 16) ahead of a bare product.
int run_int8_clear(void* p, size_t bytes, cudaStream_t stream, std::string* err);
int run_int8_rows(const Int8Rows& r, cudaStream_t stream, std::string* err);

}  // namespace tfb200
