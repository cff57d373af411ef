// Layer norm over the last axis, with its backward pass.  A row is D values; rows come as tokens (n0 x n1) of H heads,
// each head with weights of its own (H = 1: the plain layer norm).
//
//   h = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  y = h w + b
//   g = dy w,  dx = rstd (g - mean(g) - h mean(g h)),  dw = sum over tokens dy h,  db = sum over tokens dy
//
// All sums, mean and rstd are float32; y and dx are rounded once, dw and db are summed in float32 and rounded once.
// Every sum has a fixed order: the same inputs give the same bits.
#include "common.h"

namespace xl {
namespace {

constexpr int LN_BLOCK = 256;
constexpr int LN_SLICES = 512;  // most slices of the tokens that the weight's gradient is summed over first

// tokens t = i0 * n1 + i1 of x at i0 * s0 + i1 * s1 + head * sh, values contiguous
struct Rows {
  int64_t s0, s1, sh;
};
struct Shape {
  int tokens, n1, H, D;
};

__device__ __forceinline__ int64_t row_at(const Rows& r, const Shape& s, int token, int head) {
  const int i0 = s.n1 < s.tokens ? token / s.n1 : 0;
  return i0 * r.s0 + (token - i0 * s.n1) * r.s1 + head * r.sh;
}

__device__ __forceinline__ float load_param(const void* p, int64_t i, bool p32, float) { return ((const float*)p)[i]; }
template <typename T>
__device__ __forceinline__ float load_param(const void* p, int64_t i, bool p32, T) {
  return p32 ? ((const float*)p)[i] : to_f32(((const T*)p)[i]);
}

__device__ __forceinline__ float block_sum(float v, float* part) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < LN_BLOCK / 64; ++w) s += part[w];
  return s;
}

template <typename T>
__global__ __launch_bounds__(LN_BLOCK) void ln_fwd_kernel(const T* __restrict__ x, Rows xr, const void* __restrict__ w,
                                                          const void* __restrict__ b, bool p32, T* __restrict__ y,
                                                          float* __restrict__ mean, float* __restrict__ rstd, Shape s,
                                                          float eps) {
  __shared__ float part[LN_BLOCK / 64];
  const float n = (float)s.D;
  for (int64_t r = blockIdx.x; r < (int64_t)s.tokens * s.H; r += gridDim.x) {
    const int token = (int)(r / s.H), head = (int)(r - (int64_t)token * s.H);
    const T* xp = x + row_at(xr, s, token, head);
    T* yp = y + r * s.D;
    float sum = 0.f;
    for (int i = threadIdx.x; i < s.D; i += LN_BLOCK) sum += to_f32(xp[i]);
    const float mu = block_sum(sum, part) / n;
    float sq = 0.f;
    for (int i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const float d = to_f32(xp[i]) - mu;
      sq = fmaf(d, d, sq);
    }
    const float rs = 1.0f / sqrtf(block_sum(sq, part) / n + eps);
    for (int i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const int64_t c = (int64_t)head * s.D + i;
      float f = (to_f32(xp[i]) - mu) * rs;
      if (w) f *= load_param(w, c, p32, T{});
      if (b) f += load_param(b, c, p32, T{});
      yp[i] = from_f32<T>(f);
    }
    if (threadIdx.x == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(LN_BLOCK) void ln_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x, Rows xr,
                                                         const void* __restrict__ w, bool p32, const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, T* __restrict__ dx, Rows dxr,
                                                         Shape s) {
  __shared__ float part[LN_BLOCK / 64];
  const float n = (float)s.D;
  for (int64_t r = blockIdx.x; r < (int64_t)s.tokens * s.H; r += gridDim.x) {
    const int token = (int)(r / s.H), head = (int)(r - (int64_t)token * s.H);
    const T *xp = x + row_at(xr, s, token, head), *dp = dy + r * s.D;
    T* op = dx + row_at(dxr, s, token, head);
    const float mu = mean[r], rs = rstd[r];
    auto g_of = [&](int i) {
      const float d = to_f32(dp[i]);
      return w ? d * load_param(w, (int64_t)head * s.D + i, p32, T{}) : d;
    };
    float sg = 0.f, sgh = 0.f;
    for (int i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const float g = g_of(i);
      sg += g;
      sgh = fmaf(g, (to_f32(xp[i]) - mu) * rs, sgh);
    }
    const float c1 = block_sum(sg, part) / n, c2 = block_sum(sgh, part) / n;
    for (int i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const float h = (to_f32(xp[i]) - mu) * rs;
      op[i] = from_f32<T>(rs * (g_of(i) - c1 - h * c2));
    }
  }
}

// sums over one slice of the tokens: part[0][slice][c] of dy h, part[1][slice][c] of dy
template <typename T>
__global__ __launch_bounds__(LN_BLOCK) void ln_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x, Rows xr,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              float* __restrict__ part, Shape s, int slices) {
  const int64_t C = (int64_t)s.H * s.D, c = (int64_t)blockIdx.x * LN_BLOCK + threadIdx.x;
  if (c >= C) return;
  const int head = (int)(c / s.D), i = (int)(c - (int64_t)head * s.D);
  float dw = 0.f, db = 0.f;
  for (int t = blockIdx.y; t < s.tokens; t += slices) {
    const int64_t r = (int64_t)t * s.H + head;
    const float d = to_f32(dy[r * s.D + i]), h = (to_f32(x[row_at(xr, s, t, head) + i]) - mean[r]) * rstd[r];
    dw = fmaf(d, h, dw);
    db += d;
  }
  part[(int64_t)blockIdx.y * C + c] = dw;
  part[((int64_t)slices + blockIdx.y) * C + c] = db;
}

template <typename T>
__device__ __forceinline__ void store_param(void* p, int64_t i, bool p32, float v) {
  if (p32)
    ((float*)p)[i] = v;
  else
    ((T*)p)[i] = from_f32<T>(v);
}

template <typename T>
__global__ __launch_bounds__(LN_BLOCK) void ln_join_kernel(const float* __restrict__ part, void* __restrict__ dw,
                                                           void* __restrict__ db, bool p32, int64_t C, int slices) {
  const int64_t c = (int64_t)blockIdx.x * LN_BLOCK + threadIdx.x;
  if (c >= C) return;
  float a = 0.f, b = 0.f;
  for (int k = 0; k < slices; ++k) {
    a += part[k * C + c];
    b += part[(slices + k) * C + c];
  }
  if (dw) store_param<T>(dw, c, p32, a);
  if (db) store_param<T>(db, c, p32, b);
}

int slices_of(int tokens) { return tokens < 1 ? 1 : tokens < LN_SLICES ? tokens : LN_SLICES; }

unsigned grid_of(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

template <typename T>
int launch_fwd(const void* x, const Rows& xr, const void* w, const void* b, bool p32, void* y, float* mean, float* rstd,
               const Shape& s, float eps, hipStream_t st) {
  hipLaunchKernelGGL(ln_fwd_kernel<T>, dim3(grid_of((int64_t)s.tokens * s.H)), dim3(LN_BLOCK), 0, st, (const T*)x, xr, w, b,
                     p32, (T*)y, mean, rstd, s, eps);
  return check_launch("xl_layer_norm_fwd");
}

template <typename T>
int launch_bwd(const void* dy, const void* x, const Rows& xr, const void* w, bool p32, const float* mean, const float* rstd,
               void* dx, const Rows& dxr, void* dw, void* db, const Shape& s, float* part, hipStream_t st) {
  const int64_t C = (int64_t)s.H * s.D;
  const unsigned cols = (unsigned)((C + LN_BLOCK - 1) / LN_BLOCK);
  if (dx && s.tokens)
    hipLaunchKernelGGL(ln_dx_kernel<T>, dim3(grid_of((int64_t)s.tokens * s.H)), dim3(LN_BLOCK), 0, st, (const T*)dy,
                       (const T*)x, xr, w, p32, mean, rstd, (T*)dx, dxr, s);
  if (dw || db) {
    const int slices = slices_of(s.tokens);
    hipLaunchKernelGGL(ln_columns_kernel<T>, dim3(cols, (unsigned)slices), dim3(LN_BLOCK), 0, st, (const T*)dy, (const T*)x,
                       xr, mean, rstd, part, s, slices);
    hipLaunchKernelGGL(ln_join_kernel<T>, dim3(cols), dim3(LN_BLOCK), 0, st, part, dw, db, p32, C, slices);
  }
  return check_launch("xl_layer_norm_bwd");
}

// XL_OK, or the refusal of the sizes and types; s and p32 filled in
int shape_of(const char* who, int64_t n0, int64_t n1, int H, int D, int dtype, int param_dtype, Shape& s, bool& p32) {
  if (n0 < 0 || n1 < 0 || H < 1 || D < 1)
    return set_error(XL_ERR_INVALID_ARG, "%s: sizes n0=%lld n1=%lld H=%d D=%d (H and D at least 1)", who, (long long)n0,
                     (long long)n1, H, D);
  if (!dtype_ok(dtype) || (param_dtype != dtype && param_dtype != XL_DTYPE_F32))
    return set_error(XL_ERR_INVALID_ARG, "%s: dtype %d with weights of dtype %d (the same one, or float32)", who, dtype,
                     param_dtype);
  const int64_t most = 0x7fffffff;
  if (n0 > most || n1 > most || n0 * n1 > most / H || (int64_t)H * D > most)
    return set_error(XL_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows, or values per token", who);
  s = Shape{(int)(n0 * n1), (int)(n1 ? n1 : 1), H, D};
  p32 = param_dtype == XL_DTYPE_F32;
  return XL_OK;
}

Rows rows_of(const int64_t* strides, const Shape& s) {
  const int64_t C = (int64_t)s.H * s.D;
  return strides ? Rows{strides[0], strides[1], strides[2]} : Rows{C * s.n1, C, s.D};
}

}  // namespace
}  // namespace xl

extern "C" int xl_layer_norm_fwd(const void* x, const int64_t* x_strides, const void* weight, const void* bias, void* y,
                                 float* mean, float* rstd, int64_t n0, int64_t n1, int H, int D, float eps, int dtype,
                                 int param_dtype, void* stream) {
  using namespace xl;
  clear_error();
  const char* who = "xl_layer_norm_fwd";
  Shape s;
  bool p32;
  if (const int rc = shape_of(who, n0, n1, H, D, dtype, param_dtype, s, p32)) return rc;
  if (s.tokens == 0) return XL_OK;
  if (!x || !y) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (x == y) return set_error(XL_ERR_INVALID_ARG, "%s: y must not alias x", who);
  const Rows xr = rows_of(x_strides, s);
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case XL_DTYPE_F32: return launch_fwd<float>(x, xr, weight, bias, p32, y, mean, rstd, s, eps, st);
    case XL_DTYPE_BF16: return launch_fwd<bf16_t>(x, xr, weight, bias, p32, y, mean, rstd, s, eps, st);
    default: return launch_fwd<f16_t>(x, xr, weight, bias, p32, y, mean, rstd, s, eps, st);
  }
}

extern "C" size_t xl_layer_norm_bwd_workspace_size(int64_t n0, int64_t n1, int H, int D) {
  using namespace xl;
  Shape s;
  bool p32;
  if (shape_of("xl_layer_norm_bwd_workspace_size", n0, n1, H, D, XL_DTYPE_F32, XL_DTYPE_F32, s, p32)) return 0;
  return (size_t)2 * slices_of(s.tokens) * H * D * sizeof(float);
}

extern "C" int xl_layer_norm_bwd(const void* dy, const void* x, const int64_t* x_strides, const void* weight,
                                 const float* mean, const float* rstd, void* dx, const int64_t* dx_strides, void* dweight,
                                 void* dbias, int64_t n0, int64_t n1, int H, int D, int dtype, int param_dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  using namespace xl;
  clear_error();
  const char* who = "xl_layer_norm_bwd";
  Shape s;
  bool p32;
  if (const int rc = shape_of(who, n0, n1, H, D, dtype, param_dtype, s, p32)) return rc;
  if (!dx && !dweight && !dbias) return XL_OK;
  if (s.tokens && (!dy || !x || !mean || !rstd)) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (dx && (dx == dy || dx == x)) return set_error(XL_ERR_INVALID_ARG, "%s: dx must not alias dy or x", who);
  if (dweight || dbias) {
    const size_t need = xl_layer_norm_bwd_workspace_size(n0, n1, H, D);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u))
      return set_error(XL_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", who, need,
                       workspace_bytes);
  }
  const Rows xr = rows_of(x_strides, s), dxr = rows_of(dx_strides, s);
  float* part = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case XL_DTYPE_F32: return launch_bwd<float>(dy, x, xr, weight, p32, mean, rstd, dx, dxr, dweight, dbias, s, part, st);
    case XL_DTYPE_BF16: return launch_bwd<bf16_t>(dy, x, xr, weight, p32, mean, rstd, dx, dxr, dweight, dbias, s, part, st);
    default: return launch_bwd<f16_t>(dy, x, xr, weight, p32, mean, rstd, dx, dxr, dweight, dbias, s, part, st);
  }
}
