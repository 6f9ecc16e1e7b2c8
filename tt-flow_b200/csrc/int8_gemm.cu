// The int8 matrix product C = epi(A @ B^T): A [M,K] tokens, B [N,K] channels,
// both running along K, int32 sums (exact up to K = 131071), one fp32 scale per
// token and per channel applied to the finished sum.
#include "int8_math.cuh"

namespace tfb200 {

namespace {

// Any alignment: 64 x 64 tiles, 64 k values a step in shared memory, dp4a.
constexpr int kAnyTile = 64, kAnyK = 64;

__device__ __forceinline__ uint32_t load4(const int8_t* p, int k, int K) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (k + j < K) w |= static_cast<uint32_t>(static_cast<uint8_t>(p[k + j])) << (8 * j);
  return w;
}

__global__ void __launch_bounds__(256) k_int8_gemm_any(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb,
                                                       const Int8Epi e) {
  __shared__ uint32_t sa[kAnyTile][kAnyK / 4 + 1], sb[kAnyTile][kAnyK / 4 + 1];
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kAnyTile;
  const int row = threadIdx.x >> 2, seg = (threadIdx.x & 3) * 4;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.y) * kAnyTile; n0 < e.N;
       n0 += static_cast<int64_t>(gridDim.y) * kAnyTile) {
    int32_t acc[4][4] = {};
    for (int k0 = 0; k0 < e.K; k0 += kAnyK) {
      const bool a_in = m0 + row < e.M, b_in = n0 + row < e.N;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + (seg + j) * 4;
        sa[row][seg + j] = a_in ? load4(A + (m0 + row) * lda, k, e.K) : 0u;
        sb[row][seg + j] = b_in ? load4(B + (n0 + row) * ldb, k, e.K) : 0u;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kAnyK / 4; ++k) {
        int32_t a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = static_cast<int32_t>(sa[ty + 16 * i][k]);
          b[i] = static_cast<int32_t>(sb[tx + 16 * i][k]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + ty + 16 * i;
      if (m >= e.M) break;
      const float s = e.a_scale[m];
      const float factor = e.out == kInt8OutHidden ? hidden_factor(e.K, s, e.bound) : 1.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + tx + 16 * j;
        if (n < e.N) int8_store(e, acc[i][j], s, factor, m, static_cast<int>(n));
      }
    }
  }
}

}  // namespace

Int8GemmWs int8_gemm_ws(int64_t, int64_t, int64_t) { return {}; }

int run_int8_gemm(const Int8Gemm& g, cudaStream_t stream, std::string* err) {
  if (g.M > (int64_t(1) << 30) || g.N > (int64_t(1) << 30) || g.K > kInt8MaxK) {
    *err = "dimension too large";
    return -2;
  }
  const int64_t by = (g.N + kAnyTile - 1) / kAnyTile;
  const dim3 grid(static_cast<unsigned>((g.M + kAnyTile - 1) / kAnyTile), static_cast<unsigned>(by < 65535 ? by : 65535));
  k_int8_gemm_any<<<grid, 256, 0, stream>>>(g.A, g.lda, g.B, g.ldb, int8_epi(g));
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    *err = std::string("int8 gemm launch: ") + cudaGetErrorString(e);
    return -3;
  }
  count_launch();
  return 0;
}

}  // namespace tfb200
