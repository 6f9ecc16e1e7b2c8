// Rows to int8: symmetric quantisation with one scale per row, alone
// (tfb200_quantize_int8), behind RMSNorm and the residual's addition
// (tfb200_rmsnorm_int8), and of the fused MLP's hidden block.
//
//   t = x                    scale = amax / 127
//   t = (x + r) * gamma      scale = amax / 127 * 1 / sqrt(mean_k (x + r)^2 + eps)
//   q = rn(t * (127 / amax)),  amax = max_k |t|
//
// The row's 1 / rms multiplies every t alike, so it cancels in t / amax and q
// does not depend on it: the rounding to int8 acts on t itself, and 1 / rms only
// enters the scale. A row of zeros gives q = 0 and scale 0. A row that holds an
// infinity or a NaN (or whose sum of squares leaves fp32) gives q = 0 and scale
// NaN, so everything computed from it is NaN.
//
// HBM-bound: 2K bytes read and K written per row (4K and 3K with a residual; the
// hidden block is fp32, 4K and K). A row's T threads hold it in registers, so that
// it is read once and all its loads are in flight together. The arithmetic has to
// be kept short beside that: values are held as packed fp32 pairs (one f32x2
// instruction for two), and plain quantisation takes its maximum on the 16-bit
// words (the first form, which widened every value twice, took 86 us for 8192 x
// 16384 bf16 values, 58 now).
#include <algorithm>

#include "int8_math.cuh"
#include "int8_rows_span.h"

namespace tfb200 {

namespace {

constexpr int kMaxT = 512;          // threads per row
constexpr int kMaxRow = 64 * kMaxT;  // values of a row held in registers

struct RowsParams {
  int M, K;
  const void* x;
  int64_t ldx;
  const bf16* residual;
  int64_t ldr;
  const bf16* gamma;
  float eps;
  bf16* sum;
  int64_t lds;
  int8_t* q;
  int64_t ldq;
  float* scale;
  float one;  // 1 (q_pair)
  int ahead;  // prefetch_row
  uint4* zero;
  int64_t zero_vecs;
};

// Counters of the products that follow, cleared by all threads of the grid.
__device__ __forceinline__ void clear_words(uint4* zero, int64_t n) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += stride)
    zero[i] = make_uint4(0u, 0u, 0u, 0u);
}

__global__ void __launch_bounds__(256) k_int8_clear(uint4* zero, int64_t n) {
  grid_dep_wait();
  grid_dep_launch();
  clear_words(zero, n);
}

// What a row is read as: bf16, or fp32 (the hidden block).
template <int KIND>
struct RowIn {
  using type = uint16_t;
};
template <>
struct RowIn<kInt8RowsHidden> {
  using type = float;
};
__device__ __forceinline__ float in_value(uint16_t bits) { return __uint_as_float(static_cast<uint32_t>(bits) << 16); }
__device__ __forceinline__ float in_value(float v) { return v; }

// 32 bytes at a 32-byte boundary, read once.
__device__ __forceinline__ void load8_f32(const float* p, uint64_t (&v)[4]) {
  asm volatile("ld.global.L1::no_allocate.v4.b64 {%0, %1, %2, %3}, [%4];"
               : "=l"(v[0]), "=l"(v[1]), "=l"(v[2]), "=l"(v[3])
               : "l"(p)
               : "memory");
}

// max(a, |b|, |c|), NaN if one is (a is not negative).
__device__ __forceinline__ float max_abs(float a, uint64_t bc) {
  float b, c, r;
  f2_split(bc, b, c);
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

struct RowStat {
  float ss;
  uint32_t amax;
};

__device__ __forceinline__ RowStat warp_stat(RowStat s, bool squares) {
  if (squares) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.ss += __shfl_xor_sync(0xffffffffu, s.ss, o);
  }
  s.amax = __reduce_max_sync(0xffffffffu, s.amax);
  return s;
}

// The statistics over the block's threads (one row per block).
__device__ __forceinline__ RowStat block_stat(RowStat s, bool squares) {
  __shared__ float part_ss[32];
  __shared__ uint32_t part_max[32];
  s = warp_stat(s, squares);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) {
    part_ss[warp] = s.ss;
    part_max[warp] = s.amax;
  }
  __syncthreads();
  s.ss = lane < warps ? part_ss[lane] : 0.0f;
  s.amax = lane < warps ? part_max[lane] : 0u;
  return warp_stat(s, squares);
}

// The scale of a row; only the thread that stores it computes it (its root and
// divisions are as long as a warp's share of a 4096-wide row).
template <int KIND>
__device__ __forceinline__ float row_scale(const RowsParams& p, RowStat s) {
  if (s.amax >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  const float amax = __uint_as_float(s.amax);
  if (KIND != kInt8RowsNorm) return amax / 127.0f;
  const float mean = s.ss / static_cast<float>(p.K) + p.eps;
  return mean > 0.0f ? amax * (1.0f / sqrtf(mean) / 127.0f) : __uint_as_float(0x7FC00000u);
}
// Marks a row whose sum of squares left fp32 as not finite.
template <int KIND>
__device__ __forceinline__ RowStat checked(RowStat s) {
  if (KIND == kInt8RowsNorm && !(s.ss <= 3.402823466e38f)) s.amax = 0x7FC00000u;
  return s;
}

// rn of two values in the low bytes of a pair's halves. The product is rounded to
// fp32 before the integer: bf16 rows hold many values halfway between two steps,
// and 127 / amax rounded down would take them off the tie (it still takes amax / 2
// off for 20 of the 128 significands of amax). ptxas contracts a
// packed product and sum into one rounding, so the sum is a multiply-add by a 1
// that only the launch knows.
__device__ __forceinline__ uint64_t q_pair(uint64_t v, uint64_t r, uint64_t one) {
  return f2_fma(f2_mul(v, r), one, f2(12582912.0f, 12582912.0f));
}
__device__ __forceinline__ uint32_t pack4(uint64_t a, uint64_t b) {
  const uint32_t lo = __byte_perm(static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32), 0x0040);
  const uint32_t hi = __byte_perm(static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// The 16 bytes that start `half` 16-bit values into the 32 bytes w.
__device__ __forceinline__ void from_half(const uint32_t (&w)[8], int half, uint32_t (&o)[4]) {
  uint32_t a[7], b[5];
#pragma unroll
  for (int i = 0; i < 7; ++i) a[i] = half & 2 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) b[i] = half & 4 ? a[i + 2] : a[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(b[i], b[i + 1], 16 * (half & 1));
}

// How a row's values reach its threads.
//   kScalar: one at a time, T apart (any layout).
//   kVec:    8 neighbours at a time; x, residual and sum start every row on a
//            16-byte boundary, gamma and q (8) as well.
//   kShift:  8 neighbours at a time; the rows of x, residual and sum start
//            anywhere, but all three at the same place of their 16-byte granules
//            (odd widths). A thread reads two neighbouring granules and takes
//            its 8 values from them (at the ends of a padded row value by value,
//            int8_rows_span.h: 32735 x 1001 30 us padded, 26.5 read across the
//            padding; 7994 x 4099 30, 28); the sum is formed on granules. Single
//            loads took 7 times as long (8192 x 4099: 117 us against 16).
enum Mode : int { kScalar, kVec, kShift };

// Rows ahead that are brought into L2: about 12 MB of them, so that HBM is kept
// busy while blocks reduce and store.
constexpr int64_t kAheadBytes = 12 << 20;

template <typename T>
__device__ __forceinline__ void prefetch_row(const T* row, int K) {
  const uint64_t lo = (reinterpret_cast<uint64_t>(row) + 15) & ~uint64_t(15);
  const uint64_t hi = reinterpret_cast<uint64_t>(row + K) & ~uint64_t(15);
  if (hi > lo)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(lo), "r"(static_cast<uint32_t>(hi - lo))
                 : "memory");
}

// WARP: a warp per row (T = 32), else a block per row (T = blockDim.x).
// PER: values per thread.
template <int KIND, bool RES, Mode MODE, bool WARP, int PER>
__global__ void __launch_bounds__(WARP ? 128 : kMaxT,
                                  !WARP && PER == 32 && MODE == kVec && KIND != kInt8RowsNorm
                                      ? KIND == kInt8RowsHidden ? 2 : 3
                                      : 1)
    k_int8_rows(const RowsParams p) {
  // Launched with programmatic serialization: wait for the grid before (it may
  // write x or still read q), then let the next grid start its prologue.
  grid_dep_wait();
  grid_dep_launch();
  clear_words(p.zero, p.zero_vecs);
  const int T = WARP ? 32 : blockDim.x;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  // The hidden block is read from its last row, which the up projection wrote
  // last (what is left of it in L2 is read first), to its first, which the down
  // projection reads first.
  const int64_t at = WARP ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t row = KIND == kInt8RowsHidden ? p.M - 1 - at : at;
  if (WARP && at >= p.M) return;
  using In = typename RowIn<KIND>::type;
  const In* const x0 = static_cast<const In*>(p.x);
  const uint16_t* const r0 = reinterpret_cast<const uint16_t*>(p.residual);
  const In* x = x0 + row * p.ldx;
  const uint16_t* r = RES ? r0 + row * p.ldr : nullptr;
  const uint16_t* g = reinterpret_cast<const uint16_t*>(p.gamma);
  const int K = p.K;
  if (t == 0 && at + p.ahead < p.M) {
    const int64_t next = KIND == kInt8RowsHidden ? row - p.ahead : row + p.ahead;
    prefetch_row(x0 + next * p.ldx, K);
    if (RES) prefetch_row(r0 + next * p.ldr, K);
  }
  // Groups of 8 values: the first of group i, and the distance between them.
  constexpr int G = PER / 8;
  const int step = MODE == kScalar ? T : 1;
  auto first = [&](int i) { return MODE == kScalar ? t + i * 8 * T : (t + i * T) * 8; };
  // kShift: granule i holds values 8i - phase ..
  const int phase = MODE == kShift ? static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / 2) : 0;

  const RowSpan span_x = row_span(row, p.M, K, p.ldx), span_r = row_span(row, p.M, K, p.ldr);

  // Plain loads: the sum may be written over x or the residual.
  auto load8 = [&](const uint16_t* src, int k, uint32_t (&w)[4]) {
    if (MODE != kScalar && k + 8 <= K) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + k);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k0 = k + 2 * j * step, k1 = k0 + step;
        const uint32_t lo = k0 < K ? src[k0] : 0u, hi = k1 < K ? src[k1] : 0u;
        w[j] = lo | hi << 16;
      }
    }
  };
  // A granule from value k (k may be negative) of a row; one that reaches past
  // what the row's span allows is read value by value.
  auto granule = [&](const uint16_t* src, int k, const RowSpan& span, uint32_t* w) {
    const uint16_t* s = src + k;
    if (k >= K) {
      w[0] = w[1] = w[2] = w[3] = 0u;
    } else if (whole_granule(span, k)) {
      const uint4 v = *reinterpret_cast<const uint4*>(s);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = k + 2 * j >= 0 && k + 2 * j < K ? s[2 * j] : 0u;
        const uint32_t hi = k + 2 * j + 1 >= 0 && k + 2 * j + 1 < K ? s[2 * j + 1] : 0u;
        w[j] = lo | hi << 16;
      }
    }
  };
  // The row's values k .. k + 7 (0 past its end) from its granules; raw gets the
  // first of these.
  auto load_shifted = [&](const uint16_t* src, int k, const RowSpan& span, uint32_t (&w)[4], uint32_t (&raw)[4]) {
    uint32_t b[8];
    granule(src, k - phase, span, b);
    granule(src, k - phase + 8, span, b + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = b[j];
    from_half(b, phase, w);
    if (k + 8 > K) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] &= (k + 2 * j < K ? 0xFFFFu : 0u) | (k + 2 * j + 1 < K ? 0xFFFF0000u : 0u);
    }
  };
  uint32_t xw[KIND == kInt8RowsHidden ? 1 : G][4], rw[RES ? G : 1][4];
  uint32_t gw[KIND == kInt8RowsNorm && MODE == kVec ? G : 1][4];
  uint32_t sums[RES ? G : 1][4];  // bf16(x + residual); kShift: of the granule
  uint64_t v[KIND == kInt8RowsQuant ? 1 : G][4];  // t
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int k = first(i);
    if constexpr (KIND == kInt8RowsHidden) {
      if (k + 8 <= K) {
        load8_f32(x + k, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[i][j] = f2(k + 2 * j < K ? x[k + 2 * j] : 0.0f, k + 2 * j + 1 < K ? x[k + 2 * j + 1] : 0.0f);
      }
    } else if constexpr (MODE == kShift) {
      uint32_t xg[4], rg[4];
      load_shifted(x, k, span_x, xw[i], xg);
      if (RES) {
        load_shifted(r, k, span_r, rw[i], rg);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float lo, hi;
          f2_split(f2_add(f2_from_bf16x2(xg[j]), f2_from_bf16x2(rg[j])), lo, hi);
          sums[i][j] = pack_bf16(lo, hi);
        }
      }
    } else {
      load8(x, k, xw[i]);
      if (RES) load8(r, k, rw[i]);
    }
    if (KIND == kInt8RowsNorm && MODE == kVec) load8(g, k, gw[MODE == kVec ? i : 0]);
  }
  RowStat st{0.0f, 0u};
  if constexpr (KIND == kInt8RowsHidden) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = max_abs(amax, v[i][j]);
    st.amax = mag(amax);
  } else if (KIND == kInt8RowsQuant) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max_u16x2(m, xw[i][j] & 0x7FFF7FFFu);
    st.amax = max(m << 16, m & 0xFFFF0000u);
  } else {
    uint64_t ss = 0;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int k = first(i);
      if (k < K) {
        // Gamma beside the values only where it is read with them.
        if (MODE != kVec) load8(g, k, gw[0]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint64_t s = f2_from_bf16x2(xw[i][j]);
          if (RES) s = f2_add(s, f2_from_bf16x2(rw[RES ? i : 0][j]));
          ss = f2_fma(s, s, ss);
          v[i][j] = f2_mul(s, f2_from_bf16x2(gw[MODE == kVec ? i : 0][j]));
          amax = max_abs(amax, v[i][j]);
          if (RES && MODE != kShift) {
            float lo, hi;
            f2_split(s, lo, hi);
            sums[RES ? i : 0][j] = pack_bf16(lo, hi);
          }
        }
      }
    }
    float lo, hi;
    f2_split(ss, lo, hi);
    st.ss = lo + hi;
    st.amax = mag(amax);
  }
  st = WARP ? warp_stat(st, KIND == kInt8RowsNorm) : block_stat(st, KIND == kInt8RowsNorm);
  if (RES) {
    // After the row's last load: a thread's granules are its neighbour's too, and
    // the sum may be written over x or the residual.
    uint16_t* sum = reinterpret_cast<uint16_t*>(p.sum + row * p.lds);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int k = first(i) - phase;
      if (k >= K) break;
      const uint32_t(&o)[4] = sums[RES ? i : 0];
      if (MODE != kScalar && k >= 0 && k + 8 <= K) {
        *reinterpret_cast<uint4*>(sum + k) = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k + j * step >= 0 && k + j * step < K)
            sum[k + j * step] = static_cast<uint16_t>(o[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
  st = checked<KIND>(st);
  const UpScale u = up_scale(st.amax);  // q = rn(t * u.up * u.r)
  if (t == 0) p.scale[row] = row_scale<KIND>(p, st);
  int8_t* q = p.q + row * p.ldq;
  const uint64_t rr = f2(u.r, u.r), one = f2(p.one, p.one);
  auto store = [&](int i, const uint2& o) {
    const int k = first(i);
    if (MODE != kScalar && k + 8 <= K) {
      *reinterpret_cast<uint2*>(q + k) = o;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j * step < K) q[k + j * step] = static_cast<int8_t>(((j < 4 ? o.x : o.y) >> (8 * (j & 3))) & 0xFFu);
    }
  };
  auto quantise = [&](auto&& value) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      if (first(i) >= K) break;
      uint64_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = value(i, j);
      store(i, make_uint2(pack4(b[0], b[1]), pack4(b[2], b[3])));
    }
  };
  // A row of zeros, one that is not finite (both are stored as zeros) and one of
  // the smallest fp32 values go apart, so that the usual row costs nothing for
  // them.
  auto t_of = [&](int i, int j) {
    return KIND == kInt8RowsQuant ? f2_from_bf16x2(xw[i][j]) : v[KIND == kInt8RowsQuant ? 0 : i][j];
  };
  if (u.r != 0.0f && u.up == 1.0f) {
    quantise([&](int i, int j) { return q_pair(t_of(i, j), rr, one); });
  } else {
    quantise([&](int i, int j) {
      return u.r != 0.0f ? q_pair(f2_mul(t_of(i, j), f2(u.up, u.up)), rr, one) : uint64_t(0);
    });
  }
}

// Rows longer than the registers of a block (unaligned ones over 16384 values):
// the row is read twice, the second time mostly from L2.
template <int KIND, bool RES>
__global__ void __launch_bounds__(1024) k_int8_rows_long(const RowsParams p) {
  grid_dep_wait();
  grid_dep_launch();
  clear_words(p.zero, p.zero_vecs);
  const int64_t row = blockIdx.x;
  const typename RowIn<KIND>::type* x = static_cast<const typename RowIn<KIND>::type*>(p.x) + row * p.ldx;
  const uint16_t* r = RES ? reinterpret_cast<const uint16_t*>(p.residual) + row * p.ldr : nullptr;
  const uint16_t* g = reinterpret_cast<const uint16_t*>(p.gamma);
  auto value = [&](int k) {
    float s = in_value(x[k]);
    if (RES) s = __fadd_rn(s, in_value(r[k]));
    return s;
  };
  RowStat st{0.0f, 0u};
#pragma unroll 4
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    float s = value(k);
    if (KIND == kInt8RowsNorm) {
      st.ss = fmaf(s, s, st.ss);
      s = __fmul_rn(s, in_value(g[k]));
    }
    st.amax = max(st.amax, mag(s));
  }
  st = block_stat(st, KIND == kInt8RowsNorm);
  st = checked<KIND>(st);
  const UpScale u = up_scale(st.amax);  // q = rn(t * u.up * u.r)
  if (threadIdx.x == 0) p.scale[row] = row_scale<KIND>(p, st);
  // A thread reads a value of x again before it writes the sum, which may be x.
#pragma unroll 4
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    float s = value(k);
    if (RES) p.sum[row * p.lds + k] = __float2bfloat16_rn(s);
    if (KIND == kInt8RowsNorm) s = __fmul_rn(s, in_value(g[k]));
    const uint32_t b = round_bits(__fmul_rn(__fmul_rn(s, u.up), u.r));
    p.q[row * p.ldq + k] = u.r == 0.0f ? 0 : static_cast<int8_t>(b & 0xFFu);
  }
}

template <int KIND, bool RES>
cudaError_t launch_rows(RowsParams p, Mode mode, cudaStream_t s) {
  const bool hidden = KIND == kInt8RowsHidden;  // always aligned
  if (hidden) mode = kVec;
  // kShift: a granule more than the values fill.
  const int K = p.K + (mode == kShift && RES ? 8 : 0);
  const bool warp = K <= 32 * 32, wide = K > 32 * kMaxT, longer = K > kMaxRow || (wide && mode != kVec);
  // The smallest block that holds the row; with few rows, one that gives every
  // thread as few values as it can.
  const int per = p.M <= 148 ? 8 : 32;
  int T = std::min(kMaxT, std::max(128, (K + 32 * per - 1) / (32 * per) * 32));
  if (warp) T = 128;
  if (longer) T = 1024;
  const int64_t row_bytes = static_cast<int64_t>(p.K) * (RES || hidden ? 4 : 2);
  p.ahead = static_cast<int>(std::max<int64_t>(148, kAheadBytes / (row_bytes + 1)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(warp && !longer ? (p.M + 3) / 4 : p.M), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(T), 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  constexpr Mode kA = KIND == kInt8RowsHidden ? kVec : kScalar, kB = KIND == kInt8RowsHidden ? kVec : kShift;
  void (*kernel)(const RowsParams) = nullptr;
  if (longer)
    kernel = k_int8_rows_long<KIND, RES>;
  else if (wide)
    kernel = k_int8_rows<KIND, RES, kVec, false, 64>;
  else if (warp)
    kernel = mode == kVec     ? k_int8_rows<KIND, RES, kVec, true, 32>
             : mode == kShift ? k_int8_rows<KIND, RES, kB, true, 32>
                              : k_int8_rows<KIND, RES, kA, true, 32>;
  else
    kernel = mode == kVec     ? k_int8_rows<KIND, RES, kVec, false, 32>
             : mode == kShift ? k_int8_rows<KIND, RES, kB, false, 32>
                              : k_int8_rows<KIND, RES, kA, false, 32>;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

bool al(const void* p, unsigned b) { return (reinterpret_cast<uintptr_t>(p) & (b - 1)) == 0; }

}  // namespace

int run_int8_clear(void* ptr, size_t bytes, cudaStream_t stream, std::string* err) {
  const int64_t n = static_cast<int64_t>(bytes / 16);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 148)), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, k_int8_clear, static_cast<uint4*>(ptr), n);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    *err = std::string("counter clear launch: ") + cudaGetErrorString(e);
    return -3;
  }
  count_launch();
  return 0;
}

int run_int8_rows(const Int8Rows& r, cudaStream_t stream, std::string* err) {
  if (r.M > (int64_t(1) << 30) || r.K > (int64_t(1) << 30)) {
    *err = "dimension too large";
    return -2;
  }
  RowsParams p{};
  p.M = static_cast<int>(r.M);
  p.K = static_cast<int>(r.K);
  p.x = r.x;
  p.ldx = r.ldx;
  p.residual = r.residual;
  p.ldr = r.ldr;
  p.gamma = r.gamma;
  p.eps = r.eps;
  p.sum = r.sum;
  p.lds = r.lds;
  p.q = r.q;
  p.ldq = r.ldq;
  p.scale = r.scale;
  p.one = 1.0f;
  p.zero = static_cast<uint4*>(r.zero);
  p.zero_vecs = static_cast<int64_t>(r.zero_bytes / 16);
  const bool norm = r.kind == kInt8RowsNorm, res = norm && r.residual;
  // One row alone has no stride to keep aligned.
  auto rows_ok = [&](const void* b, int64_t ld) { return al(b, 16) && (ld % 8 == 0 || r.M == 1); };
  auto same_place = [&](const void* b, int64_t ld) {
    return ((reinterpret_cast<uintptr_t>(b) ^ reinterpret_cast<uintptr_t>(r.x)) & 15u) == 0 &&
           ((ld - r.ldx) % 8 == 0 || r.M == 1);
  };
  Mode mode = kScalar;
  if (al(r.q, 8) && (r.ldq % 8 == 0 || r.M == 1) && (!norm || al(r.gamma, 16))) {
    if (rows_ok(r.x, r.ldx) && (!res || (rows_ok(r.residual, r.ldr) && rows_ok(r.sum, r.lds))))
      mode = kVec;
    else if (!res || (same_place(r.residual, r.ldr) && same_place(r.sum, r.lds)))
      mode = kShift;
  }
  const cudaError_t e = r.kind == kInt8RowsHidden ? launch_rows<kInt8RowsHidden, false>(p, mode, stream)
                        : !norm                   ? launch_rows<kInt8RowsQuant, false>(p, mode, stream)
                        : res                     ? launch_rows<kInt8RowsNorm, true>(p, mode, stream)
                                                  : launch_rows<kInt8RowsNorm, false>(p, mode, stream);
  if (e != cudaSuccess) {
    *err = std::string("int8 rows launch: ") + cudaGetErrorString(e);
    return -3;
  }
  count_launch();
  return 0;
}

}  // namespace tfb200
