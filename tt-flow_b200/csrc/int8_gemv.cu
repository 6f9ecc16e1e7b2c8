// The int8 product for a handful of rows (decoding one sequence or a few). Only
// the weights' way through the SMs matters there, and the streaming kernel's
// set-up, partial-sum slots, arrivals and counters are most of a short product's
// time. Here warps read the weights straight into registers and multiply them on
// the spot; no workspace, no counters, one launch.
//
// A block of 8 warps finishes CH channels (rows of B), the warps sharing K. int32
// sums are exact in any order, so the results equal the other kernels' bit for bit.
//   k_int8_gemv_dot: one or two tokens. A warp reads 512 bytes of each of four
//     channels at a time and multiplies by dp4a; a lane's sums are added up at the
//     end. More tokens run into dp4a's latency (8 x 16384 x 4096: 24 us, 13 below).
//   k_int8_gemv_mma: up to 32 tokens, mma m16n8k32 with tokens as the 16 rows and
//     channels as the 8 columns. A lane holds 4 + 4 k values of one token and one
//     channel per instruction; which k they are is free as long as both operands
//     agree, so a lane takes 32 neighbouring bytes of each for four of them, and a
//     warp's load covers whole lines (16 bytes a lane: 5.3 us for 8 x 4096 x 4096,
//     4.8 with 32). One token: 4.7 us, k_int8_gemv_dot 4.4.
// Both want four blocks on an SM: 64 registers a thread, 2 to 4 KB in flight per
// warp (with three blocks of more registers 4096 channels no longer fit the GPU at
// once: 8 x 16384 x 4096 19 us). Copies through shared memory (cp.async) were
// slower at every size.
#include <algorithm>

#include "int8_math.cuh"

namespace tfb200 {

namespace {

constexpr int kWarps = 8, kBlocks = 4;    // warps a block, blocks an SM
constexpr int64_t kAtOnce = 148 * kBlocks;  // blocks on a B200

// 16 bytes of B, read once.
__device__ __forceinline__ uint4 load_once16(const int8_t* p, uint64_t policy) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.b32 {%0, %1, %2, %3}, [%4], %5;"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p), "l"(policy));
  return v;
}
// 32 bytes of B; WIDE: p is a multiple of 32, else of 16.
struct Bytes32 {
  uint32_t w[8];
};
template <bool WIDE>
__device__ __forceinline__ Bytes32 load_once32(const int8_t* p, uint64_t policy) {
  Bytes32 v;
  if (WIDE) {
    asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]),
                   "=r"(v.w[7])
                 : "l"(p));
  } else {
    const uint4 a = load_once16(p, policy), b = load_once16(p + 16, policy);
    v.w[0] = a.x, v.w[1] = a.y, v.w[2] = a.z, v.w[3] = a.w;
    v.w[4] = b.x, v.w[5] = b.y, v.w[6] = b.z, v.w[7] = b.w;
  }
  return v;
}
// The first n of 4 bytes, zeros behind them.
__device__ __forceinline__ uint32_t load_part(const int8_t* p, int n) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) w |= static_cast<uint32_t>(static_cast<uint8_t>(p[j])) << (8 * j);
  return w;
}

__device__ __forceinline__ void mma_16x8x32(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Sums of a block's parts of K, and its channels' scales and bias.
template <int MT, int CH, int KS>
struct Sums {
  alignas(16) int32_t v[KS][MT][CH];
  float sb[CH], bias[CH];
};

// Threads 0 .. CH - 1 fetch a channel's scale and bias each, at the start.
struct Col {
  float sb = 0.0f, bias = 0.0f;
};
template <int CH>
__device__ __forceinline__ Col load_col(const Int8Epi& e, int n0) {
  Col c;
  const int n = n0 + static_cast<int>(threadIdx.x);
  if (threadIdx.x < CH && n < e.N) {
    c.sb = e.b_scale[n];
    if (e.bias) c.bias = __bfloat162float(e.bias[n]);
  }
  return c;
}

// The rows of the next product's weights, the first bytes of which are brought
// into L2 when the block's own are on their way (0: none).
struct Next {
  const int8_t* b;
  int64_t ld;
  int rows, rows_per_block;
  uint32_t bytes;
};
__device__ __forceinline__ void prefetch_next(const Next& x) {
  for (int i = threadIdx.x; i < x.rows_per_block; i += kWarps * 32) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * x.rows_per_block + i;
    if (row < x.rows)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(x.b + row * x.ld), "r"(x.bytes) : "memory");
  }
}

// A thread finishes eight neighbouring channels of a token.
template <int MT, int CH, int KS>
__device__ __forceinline__ void finish(const Int8Epi& e, Sums<MT, CH, KS>& s, int n0, const Col& col) {
  if (threadIdx.x < CH) {
    s.sb[threadIdx.x] = col.sb;
    s.bias[threadIdx.x] = col.bias;
  }
  __syncthreads();
  const int m = threadIdx.x / (CH / 8), c = threadIdx.x % (CH / 8) * 8, n = n0 + c;
  if (m >= e.M || n >= e.N) return;
  uint32_t v[8] = {};
#pragma unroll
  for (int p = 0; p < KS; ++p)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += static_cast<uint32_t>(s.v[p][m][c + j]);
  Cols8 cols;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cols.sb[j] = f2(s.sb[c + 2 * j], s.sb[c + 2 * j + 1]);
    cols.bias[j] = f2(s.bias[c + 2 * j], s.bias[c + 2 * j + 1]);
  }
  float f[8];
  int8_values(e, v, e.a_scale[m], cols, f);
  if (e.residual) int8_residual(e, m, n, e.vec_res, f);
  int8_store(e, m, n, e.vec_out, f);
}

// MT tokens (M rounded up), four channels a warp, KS warps to a channel's K.
template <int MT, int CH>
__global__ void __launch_bounds__(kWarps * 32, kBlocks)
    k_int8_gemv_dot(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb, const Int8Epi e, int b_early,
                    const Next next) {
  constexpr int kR = 4, KS = kWarps * kR / CH, kU = 2, kStep = KS * 512;
  __shared__ Sums<MT, CH, KS> s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = warp / KS, part = warp % KS;
  const int n0 = blockIdx.x * CH;
  grid_dep_launch();
  if (!b_early) grid_dep_wait();
  // Channels and tokens past the matrices read the last one's; they are not used.
  const int8_t* b[kR];
#pragma unroll
  for (int r = 0; r < kR; ++r) b[r] = B + static_cast<int64_t>(min(n0 + grp * kR + r, e.N - 1)) * ldb;
  const int K = e.K;
  const uint64_t policy = l2_policy_evict_first();
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint4 bv[kU][kR];
  int k = (part * 32 + lane) * 16;
  auto load_b = [&] {
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int r = 0; r < kR; ++r)
        bv[u][r] = k + u * kStep + 16 <= K ? load_once16(b[r] + k + u * kStep, policy) : zero;
  };
  load_b();
  if (b_early) grid_dep_wait();  // the tokens, and the scales the launch before writes
  const Col col = load_col<CH>(e, n0);
  int32_t acc[MT][kR] = {};
  while (true) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int at = k + u * kStep;
        const uint4 a = at + 16 <= K ? *reinterpret_cast<const uint4*>(A + min(m, e.M - 1) * lda + at) : zero;
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          int32_t t = acc[m][r];
          t = __dp4a(static_cast<int>(a.x), static_cast<int>(bv[u][r].x), t);
          t = __dp4a(static_cast<int>(a.y), static_cast<int>(bv[u][r].y), t);
          t = __dp4a(static_cast<int>(a.z), static_cast<int>(bv[u][r].z), t);
          acc[m][r] = __dp4a(static_cast<int>(a.w), static_cast<int>(bv[u][r].w), t);
        }
      }
    k += kU * kStep;
    if (k - lane * 16 >= K) break;  // warp-uniform
    load_b();
  }
  prefetch_next(next);
  // The row's last K % 16 values, a lane each.
  if (part == 0 && lane < (K & 15)) {
    const int at = (K & ~15) + lane;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < kR; ++r) acc[m][r] += A[min(m, e.M - 1) * lda + at] * b[r][at];
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int32_t t = __reduce_add_sync(0xffffffffu, acc[m][r]);
      if (lane == 0) s.v[part][m][grp * kR + r] = t;
    }
  finish(e, s, n0, col);
}

// MT 8, 16 or 32, eight channels a warp.
template <int MT, int CH, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32, kBlocks)
    k_int8_gemv_mma(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb, const Int8Epi e, int b_early,
                    const Next next) {
  constexpr int KS = kWarps * 8 / CH, kU = 2, kSeg = kU * 128;
  constexpr int kTiles = (MT + 15) / 16, kHalves = MT >= 16 ? 2 : 1;  // tiles of 16 tokens, one or both halves
  __shared__ Sums<MT, CH, KS> s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = warp / KS, part = warp % KS;
  const int g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * CH;
  grid_dep_launch();
  if (!b_early) grid_dep_wait();
  const int8_t* b = B + static_cast<int64_t>(min(n0 + grp * 8 + g, e.N - 1)) * ldb;
  auto token = [&](int m) { return A + min(g + m, e.M - 1) * lda; };
  const int K = e.K;
  const uint64_t policy = l2_policy_evict_first();
  Bytes32 bv[kU];
  int k = part * kSeg + t * 32;
  auto load_b = [&] {
#pragma unroll
    for (int u = 0; u < kU; ++u)
      bv[u] = k + u * 128 + 32 <= K ? load_once32<WIDE>(b + k + u * 128, policy) : Bytes32{};
  };
  load_b();
  if (b_early) grid_dep_wait();
  const Col col = load_col<CH>(e, n0);
  int32_t acc[kTiles][4] = {};
  while (true) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = k + u * 128 + h * 16;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          uint4 x[2] = {};
#pragma unroll
          for (int i = 0; i < kHalves; ++i)
            if (k + u * 128 + 32 <= K && g + 16 * j + 8 * i < e.M)
              x[i] = *reinterpret_cast<const uint4*>(token(16 * j + 8 * i) + at);
          mma_16x8x32(acc[j], x[0].x, x[1].x, x[0].y, x[1].y, bv[u].w[4 * h], bv[u].w[4 * h + 1]);
          mma_16x8x32(acc[j], x[0].z, x[1].z, x[0].w, x[1].w, bv[u].w[4 * h + 2], bv[u].w[4 * h + 3]);
        }
      }
    k += KS * kSeg;
    if (k - t * 32 >= K) break;  // warp-uniform
    load_b();
  }
  prefetch_next(next);
  if (part == 0 && (K & 31)) {  // the row's last K % 32 values, eight a lane
    const int n = (K & 31) - t * 8, at = (K & ~31) + t * 8;
    const uint32_t w[2] = {load_part(b + at, n), load_part(b + at + 4, n - 4)};
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      uint32_t x[2][2] = {};
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        const int8_t* a = token(16 * j + 8 * i) + at;
        if (g + 16 * j + 8 * i < e.M) x[i][0] = load_part(a, n), x[i][1] = load_part(a + 4, n - 4);
      }
      mma_16x8x32(acc[j], x[0][0], x[1][0], x[0][1], x[1][1], w[0], w[1]);
    }
  }
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < kHalves; ++i)
      *reinterpret_cast<int2*>(&s.v[part][g + 16 * j + 8 * i][grp * 8 + 2 * t]) =
          make_int2(acc[j][2 * i], acc[j][2 * i + 1]);
  finish(e, s, n0, col);
}

using GemvKernel = void (*)(const int8_t*, int64_t, const int8_t*, int64_t, const Int8Epi, int, const Next);
template <int CH>
GemvKernel gemv_kernel(int64_t m, bool wide) {
  if (m <= 2) return m == 1 ? k_int8_gemv_dot<1, CH> : k_int8_gemv_dot<2, CH>;
  if (m <= 8) return wide ? k_int8_gemv_mma<8, CH, true> : k_int8_gemv_mma<8, CH, false>;
  if (m <= 16) return wide ? k_int8_gemv_mma<16, CH, true> : k_int8_gemv_mma<16, CH, false>;
  return wide ? k_int8_gemv_mma<32, CH, true> : k_int8_gemv_mma<32, CH, false>;
}

// Batches of weights that a warp reads one after the other, times the rounds in which
// the blocks fit the GPU. A warp holds 4 (8) channels for up to two (more) tokens, so
// 32 / CH (64 / CH) warps of a block share a channel's K, 1024 (256) values a batch.
int64_t steps(int64_t m, int64_t n, int64_t k, int ch) {
  const int64_t blocks = (n + ch - 1) / ch;
  const int64_t batch = m <= 2 ? 1024 * (kWarps * 4 / ch) : 256 * (kWarps * 8 / ch);
  return (k + batch - 1) / batch * ((blocks + kAtOnce - 1) / kAtOnce);
}

// Channels a block. Long rows (K >= 8192) and few channels: eight, the warps sharing K
// as widely as they can. Otherwise the fewest that fit the GPU at once, so that a
// block's warps share less of K, or fewer yet where that takes fewer steps. us with 8 /
// 16 / 32, weights rotated: 1 x 16384 x 8192 20.8 / 21.5 / 21.9, 8 x 8192 x 28672 39.9 /
// 41.6 / 41.7; 1 x 6144 x 5120 8.0 / 7.3 / 7.6, 16 x 6144 x 4096 9.6 / 8.5 / 12.9,
// 16 x 6144 x 5120 11.8 / 10.0 / 15.4; 1 x 16384 x 1024 7.2 / 5.2 / 4.6, 16 x 16384 x
// 4096 17.4 / 16.3 / 15.3, 1 x 16384 x 5120 16.1 / 14.8 / 14.0; with more channels than
// fit at once, 16 x 20480 x 4096 20.9 / - / 26.3, 16 x 24576 x 5120 29.3 / 26.7 / -, and
// where the steps mislead, 8 x 28672 x 2048 13.4 / - / 12.9, 2 x 28672 x 6144 30.4 / - /
// 31.6.
int channels(int64_t m, int64_t n, int64_t k) {
  if (k >= 8192 || n <= 8 * kAtOnce) return 8;
  int best = n <= 16 * kAtOnce ? 16 : 32;
  for (int ch = best / 2; ch >= 8; ch /= 2)
    if (steps(m, n, k, ch) < steps(m, n, k, best)) best = ch;
  return best;
}

}  // namespace

// Start and end, then the weights at the rate the kernels reach (for more tokens what
// L1 delivers of them), or a warp's batches one after the other.
double int8_gemv_us(int64_t m, int64_t n, int64_t k) {
  const double few = static_cast<double>(steps(m, n, k, channels(m, n, k)));
  const double rate = m <= 2 ? 6.7 : m <= 8 ? 5.9 : m <= 16 ? 5.0 : 2.4;  // TB/s
  const double stream = static_cast<double>(n) * static_cast<double>(k) * 1e-6 / rate;
  return (m <= 16 ? 1.2 : 2.2) + (stream > 0.7 * few ? stream : 0.7 * few);
}

// Bytes of the next product's weights that are brought into L2, which fills HBM's
// pause between the MLP's products. Whole MLP (rows x width x hidden), us, with 0 /
// 12 / 40 MB, weights rotated: 1 x 4096 x 16384 26.3 / 25.4 / 24.9, 2 x 4096 x 16384
// 28.9 / 26.6 / 26.6, 1 x 8192 x 28672 71.7 / 71.6 / 72.3, 3 x 4096 x 16384 30.0 / 29.8 /
// 30.0, 8 x 8192 x 28672 84.0 / 84.0 / 84.0, 8 x 4096 x 16384 30.3 / 30.2 / 30.3, 8 x 2048
// x 8192 14.2 / 13.8 / 13.5, 16 x 4096 x 16384 34.9 / 34.8 / 36.2, 24 x 4096 x 16384 37.1 /
// 36.9 / 36.9, 32 x 2048 x 8192 23.7 / 23.4 / 23.2.
int64_t next_bytes(int64_t m) { return static_cast<int64_t>(m <= 2 ? 40 : 12) << 20; }

int run_int8_gemv(const Int8Gemm& g, cudaStream_t stream, std::string* err) {
  const bool wide = (reinterpret_cast<uintptr_t>(g.B) & 31u) == 0 && (g.ldb % 32 == 0 || g.N == 1);
  const int ch = channels(g.M, g.N, g.K);
  const GemvKernel kernel =
      ch == 8 ? gemv_kernel<8>(g.M, wide) : ch == 16 ? gemv_kernel<16>(g.M, wide) : gemv_kernel<32>(g.M, wide);
  Next next{};
  if (g.next_b && g.next_ld % 16 == 0 && (reinterpret_cast<uintptr_t>(g.next_b) & 15u) == 0) {
    const int64_t blocks = (g.N + ch - 1) / ch;
    next.b = g.next_b;
    next.ld = g.next_ld;
    next.rows = static_cast<int>(g.next_n);
    next.rows_per_block = static_cast<int>((g.next_n + blocks - 1) / blocks);
    next.bytes = static_cast<uint32_t>(std::min(g.next_k, next_bytes(g.M) / g.next_n) / 16 * 16);
    if (next.bytes == 0) next.rows_per_block = 0;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((g.N + ch - 1) / ch), 1, 1);
  cfg.blockDim = dim3(kWarps * 32, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = a;
  cfg.numAttrs = 1;
  cudaError_t e =
      cudaLaunchKernelEx(&cfg, kernel, g.A, g.lda, g.B, g.ldb, int8_epi(g), static_cast<int>(g.b_stable), next);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    *err = std::string("int8 gemv launch: ") + cudaGetErrorString(e);
    return -3;
  }
  count_launch();
  return 0;
}

}  // namespace tfb200
