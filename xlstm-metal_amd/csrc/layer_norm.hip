// Layer norm over the last axis, with its backward pass.  A row is D values; rows come as tokens (n0 x n1) of H heads,
// each head with weights of its own (H = 1: the plain layer norm).
//
//   h = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  y = h w + b
//   g = dy w,  dx = rstd (g - mean(g) - h mean(g h)),  dw = sum over tokens dy h,  db = sum over tokens dy
//
// All sums, mean and rstd are float32; y and dx are rounded once, dw and db are summed in float32 and rounded once.
// Every sum has a fixed order: the same inputs give the same bits.
//
// Both passes are streams: x in, y out (2 values moved a value), then x, dy in, dx out (3).  A row is read once into the
// registers of a team of lanes, so mean and variance cost no second read; weights stay in registers over a workgroup's
// rows; the backward keeps the columns' sums there too and writes them once (float32, a workgroup's rows), for a short
// second launch to join.  Measured (us; torch's copy of the same bytes runs at 5.13 TB/s): 8192 x 4096 bf16 forward 23.6
// (5.7 TB/s), backward 44.7 to 47.2 (4.5 to 4.3 TB/s; x + dy -> dx as torch.add takes 36.7, without the weight's gradient
// 42.1); 8192 tokens of 8 heads of 512 forward 22.7 to 30.4 by machine, backward 45.6 to 47.8; 8 x 4096, one token each,
// 3.8 (latency).
#include <math.h>

#include <type_traits>

#include "common.h"

namespace xl {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int LN_BLOCK = 256;

// tokens t = i0 * n1 + i1 of x at i0 * s0 + i1 * s1 + head * sh, values contiguous
struct Rows {
  int64_t s0, s1, sh;
};
struct Shape {
  int tokens, n1, H, D;
};

__device__ __forceinline__ int64_t row_at(const Rows& r, const Shape& s, int token, int head) {
  const int i0 = s.n1 < s.tokens ? token / s.n1 : 0;
  return i0 * r.s0 + (int64_t)(token - i0 * s.n1) * r.s1 + head * r.sh;
}

typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
template <typename T>
using raw_at = std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4>;
// VW values by one load, at any element's address (16 bytes wide, a lane's addresses need not be multiples of it)
template <typename T, int VW>
struct Vec {
  T e[VW];
};
template <typename T, int VW>
__device__ __forceinline__ Vec<T, VW> load_vec(const T* p) {
  if constexpr (VW == 1) {
    return Vec<T, VW>{{*p}};
  } else {
    const u32x4 raw = *(const raw_at<T>*)p;
    return __builtin_bit_cast(Vec<T, VW>, raw);
  }
}
template <bool STREAM, typename T, int VW>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VW]) {
  if constexpr (VW == 1) {
    *p = from_f32<T>(f[0]);
  } else {
    u32x4 raw;
    if constexpr (is_f32<T>::value) {
      raw = __builtin_bit_cast(u32x4, f);
    } else {  // two values by one conversion
      using pair = std::conditional_t<std::is_same_v<T, f16_t>, xl_f16x2, xl_bf16x2>;
#pragma unroll
      for (int j = 0; j < VW / 2; ++j)
        raw[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((xl_f32x2{f[2 * j], f[2 * j + 1]}), pair));
    }
    if constexpr (STREAM)
      __builtin_nontemporal_store(raw, (raw_at<T>*)p);
    else
      *(raw_at<T>*)p = raw;
  }
}

template <typename T, int VW>
__device__ __forceinline__ void load_params(const void* p, int64_t i, bool p32, float (&f)[VW], float absent) {
#pragma unroll
  for (int j = 0; j < VW; ++j) f[j] = absent;
  if (!p) return;
  if (p32) {
#pragma unroll
    for (int j = 0; j < VW; ++j) f[j] = ((const float*)p)[i + j];
  } else {
    const Vec<T, VW> v = load_vec<T, VW>((const T*)p + i);
#pragma unroll
    for (int j = 0; j < VW; ++j) f[j] = to_f32(v.e[j]);
  }
}

template <typename T>
__device__ __forceinline__ void store_param(void* p, int64_t i, bool p32, float v) {
  if (p32)
    ((float*)p)[i] = v;
  else
    ((T*)p)[i] = from_f32<T>(v);
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// The sum over TL neighbouring lanes (a power of two up to 64) in every one of them, without LDS.  Partners add the
// same two values, so all lanes hold the same bits.
template <int TL>
__device__ __forceinline__ float lanes_sum(float x) {
  if constexpr (TL >= 2) x = dpp_add<0xB1>(x);    // quad_perm [1, 0, 3, 2]
  if constexpr (TL >= 4) x = dpp_add<0x4E>(x);    // quad_perm [2, 3, 0, 1]
  if constexpr (TL >= 8) x = dpp_add<0x141>(x);   // row_half_mirror
  if constexpr (TL >= 16) x = dpp_add<0x140>(x);  // row_mirror
  if constexpr (TL >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (TL >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}
// The sums of a and b over a team of TL lanes, of its own or several waves.  part: 2 x waves of the workgroup, not in
// use by the sum before (two buffers in turn: a wave is at most one sum ahead of the slowest).  The same number of
// calls in every wave of the workgroup.
template <int TL>
__device__ __forceinline__ void team_sum(float& a, float& b, float2* part) {
  a = lanes_sum<(TL < 64 ? TL : 64)>(a);
  b = lanes_sum<(TL < 64 ? TL : 64)>(b);
  if constexpr (TL > 64) {
    const int wave = threadIdx.x >> 6, first = wave & ~(TL / 64 - 1);
    if ((threadIdx.x & 63) == 0) part[wave] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < TL / 64; ++w) {
      const float2 p = part[first + w];
      a += p.x;
      b += p.y;
    }
  }
}

// What a lane holds of a row: NV vectors of VW values, vector k at column at[k].  The row's last vector is moved back to
// end with the row: its first skip[k] values are the vector before's (VW: the vector is not there).
template <int VW, int TL, int NV>
struct Columns {
  int at[NV], skip[NV];
  __device__ __forceinline__ Columns(int t, int D) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int start = (t + TL * k) * VW;
      at[k] = min(start, D - VW);
      skip[k] = min(start - at[k], VW);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {  // f(k, j) of the values that are this lane's own
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < VW; ++j)
        if (j >= skip[k]) f(k, j);
  }
};

// Teams of TL lanes, a row at a time, its values in registers (one read of x); the next row's loads are in flight while
// this one is summed.
template <typename T, int VW, int TL, int NV, int BLOCK, bool STREAM>
__global__ __launch_bounds__(BLOCK) void ln_fwd_kernel(const T* __restrict__ x, Rows xr, const void* __restrict__ w,
                                                       const void* __restrict__ b, bool p32, T* __restrict__ y,
                                                       float* __restrict__ mean, float* __restrict__ rstd, Shape s,
                                                       float eps, int slices) {
  constexpr int TEAMS = BLOCK / TL;
  __shared__ float2 part[2][BLOCK / 64];
  const int t = threadIdx.x & (TL - 1), team = threadIdx.x / TL;
  const int head = blockIdx.x % s.H, slice = blockIdx.x / s.H;
  const float n = (float)s.D;
  const Columns<VW, TL, NV> c(t, s.D);
  float wv[NV][VW], bv[NV][VW];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_params<T, VW>(w, (int64_t)head * s.D + c.at[k], p32, wv[k], 1.f);
    load_params<T, VW>(b, (int64_t)head * s.D + c.at[k], p32, bv[k], 0.f);
  }
  const int step = slices * TEAMS;
  Vec<T, VW> v[NV], ahead[NV];
  auto fetch = [&](int64_t token, Vec<T, VW>(&to)[NV]) {
    const T* p = x + row_at(xr, s, (int)min(token, (int64_t)s.tokens - 1), head);
#pragma unroll
    for (int k = 0; k < NV; ++k) to[k] = load_vec<T, VW>(p + c.at[k]);
  };
  fetch(slice * TEAMS + team, ahead);
  for (int64_t base = slice * TEAMS; base < s.tokens; base += step) {
    const int64_t token = base + team;
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = ahead[k];
    if (base + step < s.tokens) fetch(token + step, ahead);
    float sum = 0.f, none = 0.f, sq = 0.f;
    c.each([&](int k, int j) { sum += to_f32(v[k].e[j]); });
    team_sum<TL>(sum, none, part[0]);
    const float mu = sum / n;
    c.each([&](int k, int j) {
      const float d = to_f32(v[k].e[j]) - mu;
      sq = fmaf(d, d, sq);
    });
    team_sum<TL>(sq, none, part[1]);
    const float rs = 1.0f / sqrtf(sq / n + eps);
    if (token >= s.tokens) continue;  // after the workgroup's last barrier: it comes in the last round only
    const int64_t r = token * s.H + head;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (c.skip[k] >= VW) continue;
      float f[VW];
#pragma unroll
      for (int j = 0; j < VW; ++j) f[j] = fmaf((to_f32(v[k].e[j]) - mu) * rs, wv[k][j], bv[k][j]);
      store_vec<STREAM>(y + r * s.D + c.at[k], f);
    }
    if (t == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

// The backward pass of the same teams: dx of a row from its registers, and over the rows of a workgroup the sums of dy h
// and dy for every column, written once as part[slice][0 / 1][H * D].
template <typename T, int VW, int TL, int NV, int BLOCK, bool AHEAD, bool STREAM>
__global__ __launch_bounds__(BLOCK) void ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, Rows xr,
                                                       const void* __restrict__ w, bool p32, const float* __restrict__ mean,
                                                       const float* __restrict__ rstd, T* __restrict__ dx, Rows dxr,
                                                       float* __restrict__ part, Shape s, int slices) {
  constexpr int TEAMS = BLOCK / TL;
  __shared__ float2 sums[2][BLOCK / 64];
  __shared__ float cols[TEAMS > 1 ? BLOCK * NV * VW : 1];
  const int t = threadIdx.x & (TL - 1), team = threadIdx.x / TL;
  const int head = blockIdx.x % s.H, slice = blockIdx.x / s.H;
  const float n = (float)s.D;
  const Columns<VW, TL, NV> c(t, s.D);
  float wv[NV][VW], dw[NV][VW] = {}, db[NV][VW] = {};
#pragma unroll
  for (int k = 0; k < NV; ++k) load_params<T, VW>(w, (int64_t)head * s.D + c.at[k], p32, wv[k], 1.f);
  const int step = slices * TEAMS;
  Vec<T, VW> xv[NV], dv[NV], xa[NV], da[NV];
  float mu, rs, mua = 0.f, rsa = 0.f;
  auto fetch = [&](int64_t token) {
    const int at = (int)min(token, (int64_t)s.tokens - 1);
    const int64_t r = (int64_t)at * s.H + head;
    const T *xp = x + row_at(xr, s, at, head), *dp = dy + r * s.D;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      xa[k] = load_vec<T, VW>(xp + c.at[k]);
      da[k] = load_vec<T, VW>(dp + c.at[k]);
    }
    mua = mean[r];
    rsa = rstd[r];
  };
  if constexpr (AHEAD) {
    if (slice * TEAMS < s.tokens) fetch(slice * TEAMS + team);
  }
  int turn = 0;
  for (int64_t base = slice * TEAMS; base < s.tokens; base += step, turn ^= 1) {
    const int64_t token = base + team;
    if constexpr (!AHEAD) fetch(token);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      xv[k] = xa[k];
      dv[k] = da[k];
    }
    mu = mua;
    rs = rsa;
    if constexpr (AHEAD) {
      if (base + step < s.tokens) fetch(token + step);
    }
    float sg = 0.f, sgh = 0.f;
    const float own = token < s.tokens ? 1.f : 0.f;  // a team past the end adds nothing
    c.each([&](int k, int j) {
      const float d = to_f32(dv[k].e[j]), h = (to_f32(xv[k].e[j]) - mu) * rs, g = d * wv[k][j];
      sg += g;
      sgh = fmaf(g, h, sgh);
      if (own != 0.f) {
        dw[k][j] = fmaf(d, h, dw[k][j]);
        db[k][j] += d;
      }
    });
    if (!dx) continue;
    team_sum<TL>(sg, sgh, sums[turn]);
    if (token >= s.tokens) continue;
    const float c1 = sg / n, c2 = sgh / n;
    T* op = dx + row_at(dxr, s, (int)token, head);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (c.skip[k] >= VW) continue;
      float f[VW];
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        const float h = (to_f32(xv[k].e[j]) - mu) * rs;
        f[j] = rs * (to_f32(dv[k].e[j]) * wv[k][j] - c1 - h * c2);
      }
      store_vec<STREAM>(op + c.at[k], f);
    }
  }
  if (!part) return;
  const int64_t C = (int64_t)s.H * s.D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[NV][VW] = which ? db : dw;
    float* to = part + ((int64_t)slice * 2 + which) * C + (int64_t)head * s.D;
    if constexpr (TEAMS > 1) {  // the teams' sums in their order
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < VW; ++j) cols[(k * VW + j) * BLOCK + threadIdx.x] = acc[k][j];
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            float v = 0.f;
#pragma unroll 2
            for (int m = 0; m < TEAMS; ++m) v += cols[(k * VW + j) * BLOCK + m * TL + t];
            acc[k][j] = v;
          }
      }
    }
    if (team == 0) c.each([&](int k, int j) { to[c.at[k] + j] = acc[k][j]; });
  }
}

// Rows too long for registers: one workgroup a row, which is read again for each sum (from L2).
__device__ __forceinline__ float block_sum(float v, float2* part) {
  float none = 0.f;
  __syncthreads();
  team_sum<LN_BLOCK>(v, none, part);
  return v;
}

template <typename T>
__device__ __forceinline__ float param_at(const void* p, int64_t i, bool p32, float absent) {
  return !p ? absent : p32 ? ((const float*)p)[i] : to_f32(((const T*)p)[i]);
}

template <typename T>
__global__ __launch_bounds__(LN_BLOCK) void ln_fwd_long_kernel(const T* __restrict__ x, Rows xr, const void* __restrict__ w,
                                                               const void* __restrict__ b, bool p32, T* __restrict__ y,
                                                               float* __restrict__ mean, float* __restrict__ rstd, Shape s,
                                                               float eps) {
  __shared__ float2 part[LN_BLOCK / 64];
  const float n = (float)s.D;
  for (int64_t r = blockIdx.x; r < (int64_t)s.tokens * s.H; r += gridDim.x) {
    const int token = (int)(r / s.H), head = (int)(r - (int64_t)token * s.H);
    const T* xp = x + row_at(xr, s, token, head);
    T* yp = y + r * s.D;
    float sum = 0.f;
    for (int64_t i = threadIdx.x; i < s.D; i += LN_BLOCK) sum += to_f32(xp[i]);
    const float mu = block_sum(sum, part) / n;
    float sq = 0.f;
    for (int64_t i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const float d = to_f32(xp[i]) - mu;
      sq = fmaf(d, d, sq);
    }
    const float rs = 1.0f / sqrtf(block_sum(sq, part) / n + eps);
    for (int64_t i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const int64_t c = (int64_t)head * s.D + i;
      yp[i] = from_f32<T>(fmaf((to_f32(xp[i]) - mu) * rs, param_at<T>(w, c, p32, 1.f), param_at<T>(b, c, p32, 0.f)));
    }
    if (threadIdx.x == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(LN_BLOCK) void ln_dx_long_kernel(const T* __restrict__ dy, const T* __restrict__ x, Rows xr,
                                                              const void* __restrict__ w, bool p32,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              T* __restrict__ dx, Rows dxr, Shape s) {
  __shared__ float2 part[LN_BLOCK / 64];
  const float n = (float)s.D;
  for (int64_t r = blockIdx.x; r < (int64_t)s.tokens * s.H; r += gridDim.x) {
    const int token = (int)(r / s.H), head = (int)(r - (int64_t)token * s.H);
    const T *xp = x + row_at(xr, s, token, head), *dp = dy + r * s.D;
    T* op = dx + row_at(dxr, s, token, head);
    const float mu = mean[r], rs = rstd[r];
    float sg = 0.f, sgh = 0.f;
    for (int64_t i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const float g = to_f32(dp[i]) * param_at<T>(w, (int64_t)head * s.D + i, p32, 1.f);
      sg += g;
      sgh = fmaf(g, (to_f32(xp[i]) - mu) * rs, sgh);
    }
    __syncthreads();
    team_sum<LN_BLOCK>(sg, sgh, part);
    const float c1 = sg / n, c2 = sgh / n;
    for (int64_t i = threadIdx.x; i < s.D; i += LN_BLOCK) {
      const float g = to_f32(dp[i]) * param_at<T>(w, (int64_t)head * s.D + i, p32, 1.f);
      op[i] = from_f32<T>(rs * (g - c1 - (to_f32(xp[i]) - mu) * rs * c2));
    }
  }
}

// the columns' sums over one slice of the tokens, as ln_bwd_kernel writes them
template <typename T>
__global__ __launch_bounds__(LN_BLOCK) void ln_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x, Rows xr,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              float* __restrict__ part, Shape s, int slices) {
  const int64_t C = (int64_t)s.H * s.D, c = (int64_t)blockIdx.x * LN_BLOCK + threadIdx.x;
  if (c >= C) return;
  const int head = (int)(c / s.D), i = (int)(c - (int64_t)head * s.D);
  float dw = 0.f, db = 0.f;
  for (int64_t t = blockIdx.y; t < s.tokens; t += slices) {
    const int64_t r = t * s.H + head;
    const float d = to_f32(dy[r * s.D + i]), h = (to_f32(x[row_at(xr, s, (int)t, head) + i]) - mean[r]) * rstd[r];
    dw = fmaf(d, h, dw);
    db += d;
  }
  part[(int64_t)blockIdx.y * 2 * C + c] = dw;
  part[((int64_t)blockIdx.y * 2 + 1) * C + c] = db;
}

// dweight and dbias: the slices' sums, 64 columns a workgroup, its waves each a part of the slices
constexpr int LN_JOIN = 1024;
template <typename T>
__global__ __launch_bounds__(LN_JOIN) void ln_join_kernel(const float* __restrict__ part, void* __restrict__ dw,
                                                          void* __restrict__ db, bool p32, int64_t C, int slices) {
  constexpr int WAVES = LN_JOIN / 64;
  __shared__ float sums[WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.f;
  if (c < 2 * C) {
#pragma unroll 8
    for (int k = wave; k < slices; k += WAVES) v += part[(int64_t)k * 2 * C + c];
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave != 0 || c >= 2 * C) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < WAVES; ++k) v += sums[k][lane];
  if (c < C && dw) store_param<T>(dw, c, p32, v);
  if (c >= C && db) store_param<T>(db, c - C, p32, v);
}

// How a row of D values lies over lanes: teams of `lanes`, `vectors` of `width` values each, in workgroups of `block`;
// vectors 0: too long for registers.
struct Layout {
  int width, lanes, vectors, block;
  constexpr int teams() const { return vectors ? block / lanes : 1; }
};

// Forward: as many rows in a wave as fit, then a wave with up to 3 vectors a lane (no barrier: 4001 x 1333 f16 6.8 us,
// on 128 lanes 8.1), then several waves.  Backward, which holds the columns' sums besides: no third vector (18.2 us
// there, 22.5 with it), and workgroups of 512 for the wide rows, so that 256 of them write half the partial sums that 512
// of 256 threads do (us at 4096 / 8192 / 16384 columns of 64 MiB bf16: 50.4 / 53.5 / 66, with 512 workgroups 51.0 / 63.3 /
// 90); narrow rows, where many teams share a workgroup's sums, are faster the other way (16384 x 4 heads of 128: 19.9
// against 25.9).
Layout layout_of(int D, int dtype, bool backward) {
  const int vw = 16 / dtype_size(dtype), wide = backward ? 512 : LN_BLOCK;
  if (D < vw) return {1, 8, 1, LN_BLOCK};
  const int nvec = (D + vw - 1) / vw;
  if (nvec <= 64) return {vw, nvec <= 8 ? 8 : nvec <= 16 ? 16 : nvec <= 32 ? 32 : 64, 1, LN_BLOCK};
  if (nvec <= 128) return {vw, 64, 2, LN_BLOCK};
  if (nvec <= 192 && !backward) return {vw, 64, 3, LN_BLOCK};
  if (nvec <= 256) return {vw, 128, 2, wide};
  if (nvec <= 512) return {vw, 256, 2, wide};
  if (nvec <= 1024) return {vw, 256, 4, wide};
  if (nvec <= 2048) return {vw, 512, 4, 512};
  if (nvec <= 4096 && dtype == XL_DTYPE_F32) return {vw, 1024, 4, 1024};
  return {vw, LN_BLOCK, 0, LN_BLOCK};
}

// workgroups per head: enough for every token, at most `groups` in all
int slices_of(const Shape& s, const Layout& l, int groups) {
  const int64_t want = ((int64_t)s.tokens + l.teams() - 1) / l.teams(), most = groups / s.H;
  return (int)(want < 1 ? 1 : most < 1 ? 1 : want < most ? want : most);
}
// 8 waves a CU (4 of the register-filling widest rows), whose rows follow each other in registers
int bwd_slices(const Shape& s, const Layout& l) { return slices_of(s, l, l.block == LN_BLOCK ? 512 : 256); }
// every workgroup loads the weights once: 2048 x 16384 bf16 29.4 us on 512 workgroups, 34 on 1024
int fwd_slices(const Shape& s, const Layout& l) { return slices_of(s, l, l.block == LN_BLOCK ? 2048 : 512); }

unsigned grid_of(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

// f(constants of width, lanes, vectors, block)
template <typename T, bool BACKWARD, typename F>
void with_layout(const Layout& l, F&& f) {
  constexpr int VW = 16 / sizeof(T), WIDE = BACKWARD ? 512 : LN_BLOCK;
#define XL_LN(W, TL, NV, B) f(std::integral_constant<int, W>{}, std::integral_constant<int, TL>{}, \
                              std::integral_constant<int, NV>{}, std::integral_constant<int, B>{})
  if (l.width == 1) return XL_LN(1, 8, 1, LN_BLOCK);
  switch (l.lanes) {
    case 8: return XL_LN(VW, 8, 1, LN_BLOCK);
    case 16: return XL_LN(VW, 16, 1, LN_BLOCK);
    case 32: return XL_LN(VW, 32, 1, LN_BLOCK);
    case 64:
      if constexpr (!BACKWARD)
        if (l.vectors == 3) return XL_LN(VW, 64, 3, LN_BLOCK);
      return l.vectors == 1 ? XL_LN(VW, 64, 1, LN_BLOCK) : XL_LN(VW, 64, 2, LN_BLOCK);
    case 128: return XL_LN(VW, 128, 2, WIDE);
    case 256: return l.vectors == 2 ? XL_LN(VW, 256, 2, WIDE) : XL_LN(VW, 256, 4, WIDE);
    case 512: return XL_LN(VW, 512, 4, 512);
    default:
      if constexpr (is_f32<T>::value) return XL_LN(VW, 1024, 4, 1024);
  }
#undef XL_LN
}

// An output of half the L2 caches (8 of 4 MiB) or more goes past them.  us through them and past them, bf16, on one machine: forward
// 8192 x 4096 27.9 and 23.6, 8192 x 2048 14.0 and 12.7, 8192 x 1536 11.6 and 9.5; backward 50.4 and 49.3, 30.7 and 27.8,
// 27.2 and 24.3.  What is smaller stays for its reader.
template <typename T>
bool streams(const Shape& s) {
  return (int64_t)s.tokens * s.H * s.D * (int64_t)sizeof(T) >= (int64_t)16 << 20;
}

template <typename T>
int launch_fwd(const void* x, const Rows& xr, const void* w, const void* b, bool p32, void* y, float* mean, float* rstd,
               const Shape& s, float eps, int dtype, hipStream_t st) {
  const Layout l = layout_of(s.D, dtype, false);
  if (!l.vectors) {
    hipLaunchKernelGGL(ln_fwd_long_kernel<T>, dim3(grid_of((int64_t)s.tokens * s.H)), dim3(LN_BLOCK), 0, st, (const T*)x, xr,
                       w, b, p32, (T*)y, mean, rstd, s, eps);
  } else {
    const int slices = fwd_slices(s, l);
    const bool stream = streams<T>(s);
    with_layout<T, false>(l, [&](auto VW, auto TL, auto NV, auto BLOCK) {
      auto kernel = stream ? ln_fwd_kernel<T, VW.value, TL.value, NV.value, BLOCK.value, true>
                           : ln_fwd_kernel<T, VW.value, TL.value, NV.value, BLOCK.value, false>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)slices * s.H), dim3(BLOCK.value), 0, st, (const T*)x, xr, w, b, p32, (T*)y,
                         mean, rstd, s, eps, slices);
    });
  }
  return check_launch("xl_layer_norm_fwd");
}

template <typename T>
int launch_bwd(const void* dy, const void* x, const Rows& xr, const void* w, bool p32, const float* mean, const float* rstd,
               void* dx, const Rows& dxr, void* dw, void* db, const Shape& s, float* part, int dtype, hipStream_t st) {
  const int64_t C = (int64_t)s.H * s.D;
  const Layout l = layout_of(s.D, dtype, true);
  const int slices = bwd_slices(s, l);
  if (!dw && !db) part = nullptr;
  if (!l.vectors) {
    if (dx && s.tokens)
      hipLaunchKernelGGL(ln_dx_long_kernel<T>, dim3(grid_of((int64_t)s.tokens * s.H)), dim3(LN_BLOCK), 0, st, (const T*)dy,
                         (const T*)x, xr, w, p32, mean, rstd, (T*)dx, dxr, s);
    if (part)
      hipLaunchKernelGGL(ln_columns_kernel<T>, dim3((unsigned)((C + LN_BLOCK - 1) / LN_BLOCK), (unsigned)slices),
                         dim3(LN_BLOCK), 0, st, (const T*)dy, (const T*)x, xr, mean, rstd, part, s, slices);
  } else {
    with_layout<T, true>(l, [&](auto VW, auto TL, auto NV, auto BLOCK) {
      constexpr bool AHEAD = BLOCK.value < 1024;
      auto kernel = streams<T>(s) ? ln_bwd_kernel<T, VW.value, TL.value, NV.value, BLOCK.value, AHEAD, true>
                                  : ln_bwd_kernel<T, VW.value, TL.value, NV.value, BLOCK.value, AHEAD, false>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)slices * s.H), dim3(BLOCK.value), 0, st, (const T*)dy, (const T*)x, xr, w, p32,
                         mean, rstd, (T*)dx, dxr, part, s, slices);
    });
  }
  if (part)
    hipLaunchKernelGGL(ln_join_kernel<T>, dim3((unsigned)((2 * C + 63) / 64)), dim3(LN_JOIN), 0, st, part, dw, db, p32, C,
                       slices);
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
  const int64_t most = 0x7fffffff, widest = 1 << 26;  // what the grids of the column kernels take
  if (n0 > most || n1 > most || n0 * n1 > most / H || H > (1 << 20) || (int64_t)H * D > widest)
    return set_error(XL_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows, 2^20 heads or 2^26 values per token", who);
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
  if (!(eps >= 0.0f) || eps == INFINITY) return set_error(XL_ERR_INVALID_ARG, "%s: eps must be finite and >= 0", who);
  if (s.tokens == 0) return XL_OK;
  if (!x || !y) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (x == y) return set_error(XL_ERR_INVALID_ARG, "%s: y must not alias x", who);
  const Rows xr = rows_of(x_strides, s);
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case XL_DTYPE_F32: return launch_fwd<float>(x, xr, weight, bias, p32, y, mean, rstd, s, eps, dtype, st);
    case XL_DTYPE_BF16: return launch_fwd<bf16_t>(x, xr, weight, bias, p32, y, mean, rstd, s, eps, dtype, st);
    default: return launch_fwd<f16_t>(x, xr, weight, bias, p32, y, mean, rstd, s, eps, dtype, st);
  }
}

extern "C" size_t xl_layer_norm_bwd_workspace_size(int64_t n0, int64_t n1, int H, int D, int dtype) {
  using namespace xl;
  Shape s;
  bool p32;
  if (shape_of("xl_layer_norm_bwd_workspace_size", n0, n1, H, D, dtype, XL_DTYPE_F32, s, p32)) return 0;
  return (size_t)2 * bwd_slices(s, layout_of(D, dtype, true)) * H * D * sizeof(float);
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
    const size_t need = xl_layer_norm_bwd_workspace_size(n0, n1, H, D, dtype);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u))
      return set_error(XL_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", who, need,
                       workspace_bytes);
  }
  const Rows xr = rows_of(x_strides, s), dxr = rows_of(dx_strides, s);
  float* part = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case XL_DTYPE_F32: return launch_bwd<float>(dy, x, xr, weight, p32, mean, rstd, dx, dxr, dweight, dbias, s, part, dtype, st);
    case XL_DTYPE_BF16: return launch_bwd<bf16_t>(dy, x, xr, weight, p32, mean, rstd, dx, dxr, dweight, dbias, s, part, dtype, st);
    default: return launch_bwd<f16_t>(dy, x, xr, weight, p32, mean, rstd, dx, dxr, dweight, dbias, s, part, dtype, st);
  }
}
