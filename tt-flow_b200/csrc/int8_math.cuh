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
  float* hidden_max;
  int64_t ldm;
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
  e.hidden_max = g.hidden_max;
  e.ldm = g.ldm;
  return e;
}

// GELU in fp32. The int8 hidden block is quantised again right after it, so its
// error has to stay well under an int8 step of the row's largest value: the
// hardware tanh (error 2^-11 of the tanh) moved about 1 % of the hidden values
// by a step, so the tanh form is written with a sigmoid instead,
// 0.5 (1 + tanh z) = 1 / (1 + exp(-2z)), whose exponential and division are a
// few fp32 roundings off.
__device__ __forceinline__ float int8_gelu(float x, int mode) {
  if (mode == kGeluErf) return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
  if (mode == kGeluTanh) {
    const float z = 0.7978845608028654f * fmaf(0.044715f * x, x * x, x);
    return __fdividef(x, 1.0f + __expf(-2.0f * z));
  }
  return x;
}

// Largest |value| as its bits: unsigned order puts infinities and NaN on top.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// rn(v) for |v| < 2^22, half to even, in the low 16 bits: adding 1.5 * 2^23
// leaves the integer in the low bits (a conversion instruction runs at a quarter
// of the add's rate).
__device__ __forceinline__ uint32_t round_bits(float v) { return __float_as_uint(__fadd_rn(v, 12582912.0f)); }

// limit / amax as two factors: the reciprocal leaves fp32 for the smallest amax,
// which are taken up by a power of two first (exact). {0, 0} for a maximum of
// zero and for one that is not finite.
struct UpScale {
  float up, r;
};
__device__ __forceinline__ UpScale up_scale(uint32_t amax_bits, float limit) {
  const float amax = __uint_as_float(amax_bits);
  UpScale s;
  s.up = amax < 1e-30f ? 7.9228163e28f : 1.0f;
  s.r = amax_bits == 0u || amax_bits >= 0x7F800000u ? 0.0f : __fmul_rn(__frcp_rn(amax * s.up), limit);
  return s;
}

// The maximum kept for a block of the hidden values (Int8Hidden).
__device__ __forceinline__ float hidden_max(uint32_t amax_bits) {
  return __uint_as_float(amax_bits >= 0x7F800000u ? 0x7FC00000u : amax_bits);
}
// One hidden value in the low 16 bits; s = up_scale(its block's maximum, 32767).
__device__ __forceinline__ uint32_t hidden_bits(float h, UpScale s) {
  return s.r == 0.0f ? 0u : round_bits(h * s.up * s.r);
}

// acc * sa * sb, and + bias: the same roundings in every kernel and layout.
__device__ __forceinline__ float int8_scaled(int32_t acc, float sa, float sb) {
  return __fmul_rn(__fmul_rn(__int2float_rn(acc), sa), sb);
}
__device__ __forceinline__ float int8_scaled(int32_t acc, float sa, float sb, float bias) {
  return __fmaf_rn(__fmul_rn(__int2float_rn(acc), sa), sb, bias);
}

// One output value from its integer sum, without the residual.
__device__ __forceinline__ float int8_value(const Int8Epi& e, int32_t acc, float sa, int n) {
  const float v =
      e.bias ? int8_scaled(acc, sa, e.b_scale[n], __bfloat162float(e.bias[n])) : int8_scaled(acc, sa, e.b_scale[n]);
  return int8_gelu(v, e.gelu);
}

// One output value but for a hidden one, finished and stored.
__device__ __forceinline__ void int8_store(const Int8Epi& e, int32_t acc, float sa, int64_t m, int n) {
  float v = int8_value(e, acc, sa, n);
  if (e.residual) v = __fadd_rn(v, __bfloat162float(e.residual[m * e.ldr + n]));
  if (e.out == kInt8OutF32)
    static_cast<float*>(e.C)[m * e.ldc + n] = v;
  else
    static_cast<bf16*>(e.C)[m * e.ldc + n] = __float2bfloat16_rn(v);
}

}  // namespace tfb200
