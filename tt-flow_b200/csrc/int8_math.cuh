// Device arithmetic shared by the kernels of the 8-bit integer path.
#pragma once

#include "int8.h"
#include "sm100_ptx.cuh"

namespace tfb200 {

// Epilogue operands of a product (Int8Gemm without its int8 matrices).
struct Int8Epi {
  int M, N, K;
  const float* a_scale;
  const float* b_scale;
  const bf16* bias;
  int gelu;
  const bf16* residual;
  int64_t ldr;
  void* C;
  int64_t ldc;
  int out;
  // 16-byte accesses: scales and bias; the residual's rows; C's rows.
  bool vec_cols, vec_res, vec_out;
};

inline Int8Epi int8_epi(const Int8Gemm& g) {
  Int8Epi e{};
  e.M = static_cast<int>(g.M);
  e.N = static_cast<int>(g.N);
  e.K = static_cast<int>(g.K);
  e.a_scale = g.a_scale;
  e.b_scale = g.b_scale;
  e.bias = g.bias;
  e.gelu = g.gelu;
  e.residual = g.residual;
  e.ldr = g.ldr;
  e.C = g.C;
  e.ldc = g.ldc;
  e.out = g.out;
  auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  e.vec_cols = al16(g.b_scale) && (!g.bias || al16(g.bias));
  e.vec_res = al16(g.residual) && (g.ldr % 8 == 0 || g.M == 1);
  e.vec_out = al16(g.C) && (g.ldc * (g.out == kInt8OutF32 ? 4 : 2) % 16 == 0 || g.M == 1);
  return e;
}

// GELU in fp32, on packed pairs. The MLP's hidden block is quantised right after
// it, so its error has to stay well under an int8 step of the row's largest
// value: the hardware tanh (error 2^-11 of the tanh) moved about 1 % of the
// hidden values by a step. The tanh form is written with a sigmoid instead,
//   0.5 x (1 + tanh z) = x / (1 + exp(-2z)),  -2z log2(e) = x (k1 + k2 x^2),
// whose exponential (ex2.approx, 2^-22) and reciprocal (1 ulp) cost as many
// special-function instructions as the tanh and one more.
__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint64_t int8_gelu_tanh(uint64_t x) {
  // k1 = -2 log2(e) sqrt(2 / pi), k2 = 0.044715 k1
  const uint64_t k1 = f2(-2.3022081985f, -2.3022081985f), k2 = f2(-0.10294323960f, -0.10294323960f);
  float a, b;
  f2_split(f2_mul(x, f2_fma(f2_mul(x, x), k2, k1)), a, b);
  f2_split(f2_add(f2(ex2_approx(a), ex2_approx(b)), f2(1.0f, 1.0f)), a, b);
  return f2_mul(x, f2(rcp_approx(a), rcp_approx(b)));
}
__device__ __forceinline__ uint64_t int8_gelu_erf(uint64_t x) {
  float a, b;
  f2_split(x, a, b);
  a = 0.5f * a * (1.0f + erff(a * 0.70710678118654752f));
  b = 0.5f * b * (1.0f + erff(b * 0.70710678118654752f));
  return f2(a, b);
}

// Largest |value| as its bits: unsigned order puts infinities and NaN on top.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// rn(v) for |v| < 2^22, half to even, in the low 16 bits: adding 1.5 * 2^23
// leaves the integer in the low bits (a conversion instruction runs at a quarter
// of the add's rate).
__device__ __forceinline__ uint32_t round_bits(float v) { return __float_as_uint(__fadd_rn(v, 12582912.0f)); }

// 127 / amax as two factors: the reciprocal leaves fp32 for the smallest amax,
// which are taken up by a power of two first (exact). r = 0 for a maximum of zero
// and for one that is not finite.
struct UpScale {
  float up, r;
};
__device__ __forceinline__ UpScale up_scale(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits);
  UpScale s;
  s.up = amax < 1e-30f ? 7.9228163e28f : 1.0f;
  s.r = amax_bits == 0u || amax_bits >= 0x7F800000u ? 0.0f : __fmul_rn(__frcp_rn(amax * s.up), 127.0f);
  return s;
}

// acc * sa * sb + bias of two columns: the same roundings in every kernel and
// layout (without a bias it is 0).
__device__ __forceinline__ uint64_t int8_scaled(uint32_t acc0, uint32_t acc1, uint64_t sa, uint64_t sb,
                                                uint64_t bias) {
  const uint64_t v = f2(__int2float_rn(static_cast<int32_t>(acc0)), __int2float_rn(static_cast<int32_t>(acc1)));
  return f2_fma(f2_mul(v, sa), sb, bias);
}

// Eight neighbouring columns n .. n + 7 of the epilogue's operands. `vec` says
// that scales and bias start on 16-byte boundaries (n is a multiple of 8).
struct Cols8 {
  uint64_t sb[4], bias[4];  // fp32 pairs
};
__device__ __forceinline__ Cols8 int8_cols(const Int8Epi& e, int n, bool vec) {
  Cols8 c;
  if (vec && n + 8 <= e.N) {
    const float4 s0 = *reinterpret_cast<const float4*>(e.b_scale + n);
    const float4 s1 = *reinterpret_cast<const float4*>(e.b_scale + n + 4);
    const uint4 b = e.bias ? *reinterpret_cast<const uint4*>(e.bias + n) : make_uint4(0u, 0u, 0u, 0u);
    c.sb[0] = f2(s0.x, s0.y), c.sb[1] = f2(s0.z, s0.w), c.sb[2] = f2(s1.x, s1.y), c.sb[3] = f2(s1.z, s1.w);
    c.bias[0] = f2_from_bf16x2(b.x), c.bias[1] = f2_from_bf16x2(b.y);
    c.bias[2] = f2_from_bf16x2(b.z), c.bias[3] = f2_from_bf16x2(b.w);
  } else {
    float sb[8], bias[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sb[j] = n + j < e.N ? e.b_scale[n + j] : 0.0f;
      bias[j] = e.bias && n + j < e.N ? __bfloat162float(e.bias[n + j]) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c.sb[j] = f2(sb[2 * j], sb[2 * j + 1]);
      c.bias[j] = f2(bias[2 * j], bias[2 * j + 1]);
    }
  }
  return c;
}

// Scale, bias, GELU on eight columns of one row. The epilogues walk over groups
// of eight in rolled loops: with 32 columns unrolled their code did not fit the
// instruction caches, and fetching it took most of a small product's time (64 x
// 4096 x 4096: 40 us, of which the weights' stream is 3).
__device__ __forceinline__ void int8_values(const Int8Epi& e, const uint32_t (&acc)[8], float sa, const Cols8& c,
                                            float (&f)[8]) {
  uint64_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = int8_scaled(acc[2 * j], acc[2 * j + 1], f2(sa, sa), c.sb[j], c.bias[j]);
  if (e.gelu == kGeluErf) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = int8_gelu_erf(v[j]);
  } else if (e.gelu == kGeluTanh) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = int8_gelu_tanh(v[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) f2_split(v[j], f[2 * j], f[2 * j + 1]);
}

__device__ __forceinline__ void add8_bf16(const uint4& b, float (&f)[8]) {
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = __fadd_rn(f[j], (j & 1) ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]));
}

// + residual on columns n .. n + 7 of row m; `vec`: its rows start on 16-byte
// boundaries.
__device__ __forceinline__ void int8_residual(const Int8Epi& e, int64_t m, int n, bool vec, float (&f)[8]) {
  const bf16* r = e.residual + m * e.ldr + n;
  if (vec && n + 8 <= e.N) {
    add8_bf16(*reinterpret_cast<const uint4*>(r), f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n + j < e.N) f[j] = __fadd_rn(f[j], __bfloat162float(r[j]));
  }
}

__device__ __forceinline__ uint4 pack8_bf16(const float (&f)[8]) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// Columns n .. n + 7 of row m of C (bf16 or fp32); `vec`: its rows start on
// 16-byte boundaries.
__device__ __forceinline__ void int8_store(const Int8Epi& e, int64_t m, int n, bool vec, const float (&f)[8]) {
  if (e.out == kInt8OutF32) {
    float* c = static_cast<float*>(e.C) + m * e.ldc + n;
    if (vec && n + 8 <= e.N) {
      *reinterpret_cast<float4*>(c) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(c + 4) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < e.N) c[j] = f[j];
    }
  } else {
    bf16* c = static_cast<bf16*>(e.C) + m * e.ldc + n;
    if (vec && n + 8 <= e.N) {
      *reinterpret_cast<uint4*>(c) = pack8_bf16(f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < e.N) c[j] = __float2bfloat16_rn(f[j]);
    }
  }
}

}  // namespace tfb200
