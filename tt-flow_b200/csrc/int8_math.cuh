// Device arithmetic shared by the kernels of the 8-bit integer path.
#pragma once

#include <cuda_fp16.h>

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
  const float* bound;
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
  e.bound = g.bound;
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

// Power of two that brings row m's hidden values into fp16 whatever they are:
// |h| <= |u| <= 127 * 127 * K * a_scale * max |b_scale| + max |bias|, and the
// factor takes that bound to at most 32768. The products a model forms lie two
// to three orders of magnitude under the bound, where fp16 still holds 11 bits,
// eight times finer than bf16: with bf16 the second quantisation moved about
// 2 % of the hidden values by a step.
__device__ __forceinline__ float hidden_factor(int K, float a_scale, const float* bound) {
  const float u = 16129.0f * static_cast<float>(K) * fabsf(a_scale) * bound[0] + bound[1];
  if (!(u > 0.0f)) return 1.0f;  // an empty bound, or a NaN row
  const float r = fminf(fmaxf(32768.0f / u, 1.17549435e-38f), 1.2676506e30f);
  return __uint_as_float(__float_as_uint(r) & 0x7F800000u);
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

// One output value, finished and stored; `factor` is the row's hidden factor.
__device__ __forceinline__ void int8_store(const Int8Epi& e, int32_t acc, float sa, float factor, int64_t m, int n) {
  float v = int8_value(e, acc, sa, n);
  if (e.residual) v = __fadd_rn(v, __bfloat162float(e.residual[m * e.ldr + n]));
  if (e.out == kInt8OutF32)
    static_cast<float*>(e.C)[m * e.ldc + n] = v;
  else if (e.out == kInt8OutBf16)
    static_cast<bf16*>(e.C)[m * e.ldc + n] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(e.C)[m * e.ldc + n] = __float2half_rn(v * factor);
}

}  // namespace tfb200
