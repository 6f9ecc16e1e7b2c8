// C ABI of the 8-bit integer path (declared in include/tfb200.h): argument
// checks, workspace layout and dispatch.
#include <string>

#include "../../include/tfb200.h"
#include "int8.h"

namespace tfb200 {

namespace {

constexpr int64_t kMaxDim = int64_t(1) << 30;
constexpr size_t kTooBig = ~size_t(0);

size_t al256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }
int64_t ld16(int64_t k) { return (k + 15) / 16 * 16; }
int64_t ld_hidden(int64_t h) { return (h + 7) / 8 * 8; }  // fp32 rows on 32-byte boundaries

int fail(int code, const char* fn, const std::string& msg) {
  set_last_error(std::string(fn) + ": " + msg);
  return code;
}

// Runs an entry point's body; nothing it throws (an allocation in a message)
// crosses the C boundary.
template <typename F>
int guarded(F&& body) {
  try {
    return body();
  } catch (...) {
    return TFB200_ECUDA;
  }
}

bool mat_ok(const tfb200_mat* m, const char* name, int32_t dtype, std::string* err) {
  static const char* const names[] = {"TFB200_BF16", "TFB200_F32", "TFB200_I8"};
  if (!m) {
    *err = std::string(name) + ": null descriptor";
  } else if (m->dtype != dtype) {
    *err = std::string(name) + ": dtype must be " + names[dtype];
  } else if (m->rows < 0 || m->cols < 0) {
    *err = std::string(name) + ": negative shape";
  } else if (m->rows > kMaxDim || m->cols > kMaxDim) {
    *err = std::string(name) + ": dimension above 2^30";
  } else if (m->ld < m->cols || m->ld < 1) {
    *err = std::string(name) + ": leading dimension smaller than the column count";
  } else if (!m->data && m->rows > 0 && m->cols > 0) {
    *err = std::string(name) + ": null data";
  } else if (dtype != TFB200_I8 && (reinterpret_cast<uintptr_t>(m->data) & (dtype == TFB200_F32 ? 3u : 1u))) {
    *err = std::string(name) + ": data not aligned to its element";
  } else {
    return true;
  }
  return false;
}

// gamma and bias (2 bytes), scales (4): null is the caller's to judge.
bool vec_ok(const void* p, unsigned bytes, const char* name, std::string* err) {
  if (!(reinterpret_cast<uintptr_t>(p) & (bytes - 1))) return true;
  *err = std::string(name) + ": not aligned to its element";
  return false;
}

bool same_shape(const tfb200_mat* a, const tfb200_mat* b) { return a->rows == b->rows && a->cols == b->cols; }

const bf16* as_bf16(const void* p) { return static_cast<const bf16*>(p); }

// Workspace of the fused calls: int8 rows and their scales, (MLP: the hidden
// block in fp32, its int8 form and scales), then each product's region, whose
// counters the rows launch ahead of it clears.
struct Layout {
  size_t q = 0, scale = 0, hidden = 0, hq = 0, hscale = 0, up = 0, down = 0, up_clear = 0, down_clear = 0,
         total = 0;
};

Layout layout(int64_t m, int64_t k, int64_t h, int64_t n) {
  Layout l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += al256(bytes);
    return here;
  };
  const size_t rows = static_cast<size_t>(m);
  l.q = take(rows * ld16(k));
  l.scale = take(rows * 4);
  if (h > 0) {
    l.hidden = take(rows * ld_hidden(h) * sizeof(float));
    l.hq = take(rows * ld16(h));
    l.hscale = take(rows * 4);
  }
  const Int8GemmWs up = int8_gemm_ws(m, h > 0 ? h : n, k);
  l.up = take(up.total);
  l.up_clear = up.clear_bytes;
  if (h > 0) {
    const Int8GemmWs down = int8_gemm_ws(m, n, h);
    l.down = take(down.total);
    l.down_clear = down.clear_bytes;
  }
  l.total = at;
  return l;
}

bool dims_ok(int64_t m, int64_t k, int64_t n) { return m <= kMaxDim && k <= kMaxDim && n <= kMaxDim; }

int ws_check(const char* fn, const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need))
    return fail(TFB200_EWORKSPACE, fn, "workspace smaller than the " + std::to_string(need) + " bytes this call needs");
  if (need && (reinterpret_cast<uintptr_t>(ws) & 255u))
    return fail(TFB200_EWORKSPACE, fn, "workspace must be 256-byte aligned");
  return TFB200_OK;
}

int gelu_of(int mode) {
  return mode == TFB200_GELU_ERF ? kGeluErf : mode == TFB200_GELU_TANH ? kGeluTanh : kGeluNone;
}

const char kLongK[] = "inner dimension above 131071: the int32 sums could overflow";

}  // namespace

}  // namespace tfb200

using namespace tfb200;

extern "C" {

int tfb200_quantize_int8(const tfb200_mat* x, tfb200_mat* q, float* scale, void* stream) {
  static const char fn[] = "tfb200_quantize_int8";
  return guarded([&] {
    std::string err;
    if (!mat_ok(x, "x", TFB200_BF16, &err) || !mat_ok(q, "q", TFB200_I8, &err) || !vec_ok(scale, 4, "scale", &err))
      return fail(TFB200_EINVAL, fn, err);
    if (!same_shape(x, q)) return fail(TFB200_EINVAL, fn, "q must have the shape of x");
    if (x->rows == 0) return static_cast<int>(TFB200_OK);
    if (!scale) return fail(TFB200_EINVAL, fn, "null scale");
    Int8Rows r;
    r.M = x->rows;
    r.K = x->cols;
    r.x = x->data;
    r.ldx = x->ld;
    r.q = static_cast<int8_t*>(q->data);
    r.ldq = q->ld;
    r.scale = scale;
    const int rc = run_int8_rows(r, static_cast<cudaStream_t>(stream), &err);
    return rc ? fail(rc, fn, err) : static_cast<int>(TFB200_OK);
  });
}

int tfb200_rmsnorm_int8(const tfb200_mat* x, const tfb200_mat* residual, const void* gamma, float eps,
                        tfb200_mat* sum, tfb200_mat* q, float* scale, void* stream) {
  static const char fn[] = "tfb200_rmsnorm_int8";
  return guarded([&] {
    std::string err;
    if (!mat_ok(x, "x", TFB200_BF16, &err) || !mat_ok(q, "q", TFB200_I8, &err) ||
        !vec_ok(gamma, 2, "gamma", &err) || !vec_ok(scale, 4, "scale", &err) ||
        (residual && (!mat_ok(residual, "residual", TFB200_BF16, &err) || !mat_ok(sum, "sum", TFB200_BF16, &err))))
      return fail(TFB200_EINVAL, fn, err);
    if (!same_shape(x, q) || (residual && (!same_shape(x, residual) || !same_shape(x, sum))))
      return fail(TFB200_EINVAL, fn, "residual, sum and q must have the shape of x");
    if (!residual && sum) return fail(TFB200_EINVAL, fn, "a sum without a residual");
    if (!(eps >= 0.0f)) return fail(TFB200_EINVAL, fn, "eps must be >= 0");
    if (x->rows == 0) return static_cast<int>(TFB200_OK);
    if (x->cols == 0) return fail(TFB200_EINVAL, fn, "RMSNorm over an empty dimension");
    if (!gamma || !scale) return fail(TFB200_EINVAL, fn, "null gamma or scale");
    Int8Rows r;
    r.kind = kInt8RowsNorm;
    r.M = x->rows;
    r.K = x->cols;
    r.x = x->data;
    r.ldx = x->ld;
    r.gamma = as_bf16(gamma);
    r.eps = eps;
    if (residual) {
      r.residual = as_bf16(residual->data);
      r.ldr = residual->ld;
      r.sum = static_cast<bf16*>(sum->data);
      r.lds = sum->ld;
    }
    r.q = static_cast<int8_t*>(q->data);
    r.ldq = q->ld;
    r.scale = scale;
    const int rc = run_int8_rows(r, static_cast<cudaStream_t>(stream), &err);
    return rc ? fail(rc, fn, err) : static_cast<int>(TFB200_OK);
  });
}

size_t tfb200_matmul_int8_workspace_size(int64_t m, int64_t k, int64_t n) {
  if (m <= 0 || k <= 0 || n <= 0) return 0;
  if (!dims_ok(m, k, n)) return kTooBig;
  return int8_gemm_ws(m, n, k).total;
}

int tfb200_matmul_int8(const tfb200_mat* a, const float* a_scale, const tfb200_mat* b, const float* b_scale,
                       const void* bias, int gelu_mode, const tfb200_mat* residual, tfb200_mat* c, void* stream,
                       void* workspace, size_t workspace_bytes) {
  static const char fn[] = "tfb200_matmul_int8";
  return guarded([&] {
    std::string err;
    const bool f32 = c && c->dtype == TFB200_F32;
    if (!mat_ok(a, "a", TFB200_I8, &err) || !mat_ok(b, "b", TFB200_I8, &err) ||
        !vec_ok(a_scale, 4, "a_scale", &err) || !vec_ok(b_scale, 4, "b_scale", &err) ||
        !vec_ok(bias, 2, "bias", &err) || !mat_ok(c, "c", f32 ? TFB200_F32 : TFB200_BF16, &err) ||
        (residual && !mat_ok(residual, "residual", TFB200_BF16, &err)))
      return fail(TFB200_EINVAL, fn, err);
    if (a->cols != b->cols || c->rows != a->rows || c->cols != b->rows || (residual && !same_shape(residual, c)))
      return fail(TFB200_EINVAL, fn, "shapes do not agree (A[M,K], B[N,K], R[M,N] -> C[M,N])");
    if (gelu_mode != TFB200_GELU_NONE && gelu_mode != TFB200_GELU_ERF && gelu_mode != TFB200_GELU_TANH)
      return fail(TFB200_EINVAL, fn, "gelu_mode must be TFB200_GELU_NONE, TFB200_GELU_ERF or TFB200_GELU_TANH");
    if (a->cols > kInt8MaxK) return fail(TFB200_EUNSUPPORTED, fn, kLongK);
    if (c->rows == 0 || c->cols == 0) return static_cast<int>(TFB200_OK);
    if (!a_scale || !b_scale) return fail(TFB200_EINVAL, fn, "null scales");
    const size_t need = tfb200_matmul_int8_workspace_size(a->rows, a->cols, b->rows);
    if (const int rc = ws_check(fn, workspace, workspace_bytes, need)) return rc;
    Int8Gemm g;
    g.M = a->rows;
    g.N = b->rows;
    g.K = a->cols;
    g.A = static_cast<const int8_t*>(a->data);
    g.lda = a->ld;
    g.B = static_cast<const int8_t*>(b->data);
    g.ldb = b->ld;
    g.a_scale = a_scale;
    g.b_scale = b_scale;
    g.bias = as_bf16(bias);
    g.gelu = gelu_of(gelu_mode);
    if (residual) {
      g.residual = as_bf16(residual->data);
      g.ldr = residual->ld;
    }
    g.C = c->data;
    g.ldc = c->ld;
    g.out = f32 ? kInt8OutF32 : kInt8OutBf16;
    g.ws = workspace;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const size_t clear = int8_gemm_ws(g.M, g.N, g.K).clear_bytes;
    if (clear) {
      const int rc = run_int8_clear(workspace, clear, s, &err);
      if (rc) return fail(rc, fn, err);
      g.a_stable = g.b_stable = true;  // the clear touches only the workspace
    }
    const int rc = run_int8_gemm(g, s, &err);
    return rc ? fail(rc, fn, err) : static_cast<int>(TFB200_OK);
  });
}

size_t tfb200_fused_rmsnorm_matmul_int8_workspace_size(int64_t m, int64_t k, int64_t n) {
  if (m <= 0 || k <= 0 || n <= 0) return 0;
  if (!dims_ok(m, k, n)) return kTooBig;
  return layout(m, k, 0, n).total;
}

int tfb200_fused_rmsnorm_matmul_int8(const tfb200_mat* x, const void* gamma, const tfb200_mat* w,
                                     const float* w_scale, float eps, tfb200_mat* y, void* stream, void* workspace,
                                     size_t workspace_bytes) {
  static const char fn[] = "tfb200_fused_rmsnorm_matmul_int8";
  return guarded([&] {
    std::string err;
    if (!mat_ok(x, "x", TFB200_BF16, &err) || !mat_ok(w, "w", TFB200_I8, &err) ||
        !mat_ok(y, "y", TFB200_BF16, &err) || !vec_ok(gamma, 2, "gamma", &err) || !vec_ok(w_scale, 4, "w_scale", &err))
      return fail(TFB200_EINVAL, fn, err);
    const int64_t M = x->rows, K = x->cols, N = w->rows;
    if (w->cols != K || y->rows != M || y->cols != N)
      return fail(TFB200_EINVAL, fn, "shapes do not agree (X[M,K], W[N,K] -> Y[M,N])");
    if (!(eps >= 0.0f)) return fail(TFB200_EINVAL, fn, "eps must be >= 0");
    if (K > kInt8MaxK) return fail(TFB200_EUNSUPPORTED, fn, kLongK);
    if (M == 0 || N == 0) return static_cast<int>(TFB200_OK);
    if (K == 0) return fail(TFB200_EINVAL, fn, "RMSNorm over an empty dimension");
    if (!gamma || !w_scale) return fail(TFB200_EINVAL, fn, "null gamma or w_scale");
    const Layout l = layout(M, K, 0, N);
    if (const int rc = ws_check(fn, workspace, workspace_bytes, l.total)) return rc;
    char* ws = static_cast<char*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Int8Rows r;
    r.kind = kInt8RowsNorm;
    r.M = M;
    r.K = K;
    r.x = x->data;
    r.ldx = x->ld;
    r.gamma = as_bf16(gamma);
    r.eps = eps;
    r.q = reinterpret_cast<int8_t*>(ws + l.q);
    r.ldq = ld16(K);
    r.scale = reinterpret_cast<float*>(ws + l.scale);
    r.zero = ws + l.up;
    r.zero_bytes = l.up_clear;
    int rc = run_int8_rows(r, s, &err);
    if (rc) return fail(rc, fn, err);
    Int8Gemm g;
    g.M = M;
    g.N = N;
    g.K = K;
    g.A = r.q;
    g.lda = r.ldq;
    g.B = static_cast<const int8_t*>(w->data);
    g.ldb = w->ld;
    g.a_scale = r.scale;
    g.b_scale = w_scale;
    g.C = y->data;
    g.ldc = y->ld;
    g.ws = ws + l.up;
    g.b_stable = true;
    rc = run_int8_gemm(g, s, &err);
    return rc ? fail(rc, fn, err) : static_cast<int>(TFB200_OK);
  });
}

size_t tfb200_fused_mlp_int8_workspace_size(int64_t m, int64_t k, int64_t h, int64_t n) {
  if (m <= 0 || k <= 0 || h <= 0 || n <= 0) return 0;
  if (!dims_ok(m, k, n) || h > kMaxDim) return kTooBig;
  return layout(m, k, h, n).total;
}

int tfb200_fused_mlp_int8(const tfb200_mat* x, const void* gamma, const tfb200_mat* w1, const float* w1_scale,
                          const void* b1, const tfb200_mat* w2, const float* w2_scale, const tfb200_mat* residual,
                          float eps, int gelu_mode, tfb200_mat* y, void* stream, void* workspace,
                          size_t workspace_bytes) {
  static const char fn[] = "tfb200_fused_mlp_int8";
  return guarded([&] {
    std::string err;
    if (!mat_ok(x, "x", TFB200_BF16, &err) || !mat_ok(w1, "w1", TFB200_I8, &err) ||
        !mat_ok(w2, "w2", TFB200_I8, &err) || !mat_ok(residual, "residual", TFB200_BF16, &err) ||
        !mat_ok(y, "y", TFB200_BF16, &err) || !vec_ok(gamma, 2, "gamma", &err) || !vec_ok(b1, 2, "b1", &err) ||
        !vec_ok(w1_scale, 4, "w1_scale", &err) || !vec_ok(w2_scale, 4, "w2_scale", &err))
      return fail(TFB200_EINVAL, fn, err);
    const int64_t M = x->rows, K = x->cols, H = w1->rows, N = w2->rows;
    if (w1->cols != K || w2->cols != H || y->rows != M || y->cols != N || !same_shape(residual, y))
      return fail(TFB200_EINVAL, fn, "shapes do not agree (X[M,K], W1[H,K], W2[N,H], R[M,N] -> Y[M,N])");
    if (gelu_mode != TFB200_GELU_ERF && gelu_mode != TFB200_GELU_TANH)
      return fail(TFB200_EINVAL, fn, "gelu_mode must be TFB200_GELU_ERF or TFB200_GELU_TANH");
    if (!(eps >= 0.0f)) return fail(TFB200_EINVAL, fn, "eps must be >= 0");
    if (K > kInt8MaxK || H > kInt8MaxK) return fail(TFB200_EUNSUPPORTED, fn, kLongK);
    if (M == 0 || N == 0) return static_cast<int>(TFB200_OK);
    if (K == 0) return fail(TFB200_EINVAL, fn, "RMSNorm over an empty dimension");
    if (H == 0) return fail(TFB200_EUNSUPPORTED, fn, "empty hidden dimension");
    if (!gamma || !w1_scale || !w2_scale) return fail(TFB200_EINVAL, fn, "null gamma, w1_scale or w2_scale");
    const Layout l = layout(M, K, H, N);
    if (const int rc = ws_check(fn, workspace, workspace_bytes, l.total)) return rc;
    char* ws = static_cast<char*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Norm and quantisation of the tokens; the same launch clears the up
    // projection's counters.
    Int8Rows r;
    r.kind = kInt8RowsNorm;
    r.M = M;
    r.K = K;
    r.x = x->data;
    r.ldx = x->ld;
    r.gamma = as_bf16(gamma);
    r.eps = eps;
    r.q = reinterpret_cast<int8_t*>(ws + l.q);
    r.ldq = ld16(K);
    r.scale = reinterpret_cast<float*>(ws + l.scale);
    r.zero = ws + l.up;
    r.zero_bytes = l.up_clear;
    int rc = run_int8_rows(r, s, &err);
    if (rc) return fail(rc, fn, err);
    Int8Gemm up;
    up.M = M;
    up.N = H;
    up.K = K;
    up.A = r.q;
    up.lda = r.ldq;
    up.B = static_cast<const int8_t*>(w1->data);
    up.ldb = w1->ld;
    up.a_scale = r.scale;
    up.b_scale = w1_scale;
    up.bias = as_bf16(b1);
    up.gelu = gelu_of(gelu_mode);
    up.C = ws + l.hidden;
    up.ldc = ld_hidden(H);
    up.out = kInt8OutF32;
    up.ws = ws + l.up;
    up.b_stable = true;
    up.next_b = static_cast<const int8_t*>(w2->data);
    up.next_n = N;
    up.next_k = H;
    up.next_ld = w2->ld;
    rc = run_int8_gemm(up, s, &err);
    if (rc) return fail(rc, fn, "up projection: " + err);
    // The hidden block, per token.
    Int8Rows hr;
    hr.kind = kInt8RowsHidden;
    hr.M = M;
    hr.K = H;
    hr.x = up.C;
    hr.ldx = up.ldc;
    hr.q = reinterpret_cast<int8_t*>(ws + l.hq);
    hr.ldq = ld16(H);
    hr.scale = reinterpret_cast<float*>(ws + l.hscale);
    hr.zero = ws + l.down;
    hr.zero_bytes = l.down_clear;
    rc = run_int8_rows(hr, s, &err);
    if (rc) return fail(rc, fn, "hidden block: " + err);
    Int8Gemm down;
    down.M = M;
    down.N = N;
    down.K = H;
    down.A = hr.q;
    down.lda = hr.ldq;
    down.B = static_cast<const int8_t*>(w2->data);
    down.ldb = w2->ld;
    down.a_scale = hr.scale;
    down.b_scale = w2_scale;
    down.residual = as_bf16(residual->data);
    down.ldr = residual->ld;
    down.C = y->data;
    down.ldc = y->ld;
    down.ws = ws + l.down;
    down.b_stable = true;
    rc = run_int8_gemm(down, s, &err);
    return rc ? fail(rc, fn, "down projection: " + err) : static_cast<int>(TFB200_OK);
  });
}

}  // extern "C"
