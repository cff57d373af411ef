// Gated delta rule token by token (decode steps, a few drafted tokens):
//
//   S = a S + k d^T,  d = beta (v - a S^T k),  h = scale S^T q,  a = exp(g)
//
// A workgroup takes 32 columns of a head's state through all tokens, in float32 registers: 4 waves x 8 lane groups share
// the rows, a lane holds 4 columns of every 32nd row.  S^T k and S^T q of the state before the token are summed
// together (h = scale (a S^T q + (q.k) d)), so a token costs one reduction and one barrier.  One token is bound by the state's
// bytes, in and out once.
#include "delta.h"

namespace xl {
namespace delta {
namespace {

constexpr int COLS = 32, RWAVES = 4;

struct RecArgs {
  const void *q, *k, *v, *g, *beta;
  const float* c0;
  void* h;
  float* c_last;
  int NH, group, S, DK, DV;
  float scale;
  bool wide;  // 16-byte accesses to the state
};

template <typename T, typename G, int NI>
__global__ __launch_bounds__(256) void delta_recurrent_kernel(RecArgs p) {
  __shared__ float qk_s[2][2][MAX_DQK];
  __shared__ float sums[2][RWAVES][2][COLS];
  __shared__ float dots[2][RWAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lg = lane >> 3;
  const int slices = (p.DV + COLS - 1) / COLS;
  const int all = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int bh = all / slices, col = (all - bh * slices) * COLS + (lane & 7) * 4;
  const int b = bh / p.NH, h = bh - b * p.NH, bhk = b * (p.NH / p.group) + h / p.group;
  const T* q = (const T*)p.q + (int64_t)bhk * p.S * p.DK;
  const T* k = (const T*)p.k + (int64_t)bhk * p.S * p.DK;
  const T* v = (const T*)p.v + (int64_t)bh * p.S * p.DV;
  T* ho = (T*)p.h + (int64_t)bh * p.S * p.DV;
  const G *gp = (const G*)p.g + (int64_t)bh * p.S, *bp = (const G*)p.beta + (int64_t)bh * p.S;
  const int64_t state = (int64_t)bh * p.DK * p.DV;
  const int row0 = wave * 8 + lg;
  const bool whole = p.wide && col < p.DV;  // a multiple of 4 columns

  f32x4 st[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = row0 + 32 * i;
    st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (p.c0 && r < p.DK) {
      const float* from = p.c0 + state + (int64_t)r * p.DV + col;
      if (whole) {
        st[i] = __builtin_nontemporal_load((const f32x4*)from);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.DV) st[i][e] = from[e];
      }
    }
  }
  float qn = 0.f, kn = 0.f;  // thread tid has value tid of the next token's q and k
  if (tid < p.DK && p.S > 0) {
    qn = to_f32(q[tid]);
    kn = to_f32(k[tid]);
  }
  if (tid < MAX_DQK) {
    qk_s[0][0][tid] = qn;
    qk_s[0][1][tid] = kn;
  }
  __syncthreads();
  for (int t = 0; t < p.S; ++t) {
    const int at = t & 1;
    if (t + 1 < p.S && tid < p.DK) {
      qn = to_f32(q[(int64_t)(t + 1) * p.DK + tid]);
      kn = to_f32(k[(int64_t)(t + 1) * p.DK + tid]);
    }
    const float a = expf(to_f32(gp[t])), beta = to_f32(bp[t]);
    float vt[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) vt[e] = col + e < p.DV ? to_f32(v[(int64_t)t * p.DV + col + e]) : 0.f;
    f32x4 ks = {0.f, 0.f, 0.f, 0.f}, qs = {0.f, 0.f, 0.f, 0.f};
    float kk[NI], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float qi = qk_s[at][0][row0 + 32 * i];
      kk[i] = qk_s[at][1][row0 + 32 * i];
      dot = fmaf(qi, kk[i], dot);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] = fmaf(kk[i], st[i][e], ks[e]);
        qs[e] = fmaf(qi, st[i][e], qs[e]);
      }
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] += __shfl_xor(ks[e], o, 64);
        qs[e] += __shfl_xor(qs[e], o, 64);
      }
      dot += __shfl_xor(dot, o, 64);
    }
    if (lane < 8) {
      *(f32x4*)&sums[at][wave][0][lane * 4] = ks;
      *(f32x4*)&sums[at][wave][1][lane * 4] = qs;
      if (lane == 0) dots[at][wave] = dot;
    }
    if (tid < MAX_DQK) {
      qk_s[at ^ 1][0][tid] = qn;
      qk_s[at ^ 1][1][tid] = kn;
    }
    __syncthreads();
    ks = qs = f32x4{0.f, 0.f, 0.f, 0.f};
    dot = 0.f;
#pragma unroll
    for (int w = 0; w < RWAVES; ++w) {
      ks += *(const f32x4*)&sums[at][w][0][(lane & 7) * 4];
      qs += *(const f32x4*)&sums[at][w][1][(lane & 7) * 4];
      dot += dots[at][w];
    }
    f32x4 d;
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = beta * (vt[e] - a * ks[e]);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) st[i][e] = fmaf(kk[i], d[e], a * st[i][e]);
    if (wave == 0 && lg == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.DV) ho[(int64_t)t * p.DV + col + e] = from_f32<T>(p.scale * fmaf(dot, d[e], a * qs[e]));
    }
  }
  if (!p.c_last) return;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = row0 + 32 * i;
    if (r >= p.DK) continue;
    float* to = p.c_last + state + (int64_t)r * p.DV + col;
    if (whole) {
      *(f32x4*)to = st[i];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.DV) to[e] = st[i][e];
    }
  }
}

template <typename T, typename G>
const void* pick(int DK) {
  return DK <= 64 ? (const void*)delta_recurrent_kernel<T, G, 2> : DK <= 128 ? (const void*)delta_recurrent_kernel<T, G, 4>
                                                                             : (const void*)delta_recurrent_kernel<T, G, 8>;
}

}  // namespace

int check_shape(const char* who, const Shape& s) {
  if (s.B < 1 || s.NH < 1 || s.NHK < 1 || s.S < 0 || s.DK < 1 || s.DV < 1)
    return set_error(XL_ERR_INVALID_ARG, "%s: B, NH, NHK, DQK and DV must be positive and S not negative", who);
  if (s.NH % s.NHK != 0) return set_error(XL_ERR_INVALID_ARG, "%s: NH %d is not a multiple of NHK %d", who, s.NH, s.NHK);
  if (!dtype_ok(s.dtype) || !dtype_ok(s.dtype_gates)) return set_error(XL_ERR_INVALID_ARG, "%s: bad dtype", who);
  if (s.DK > MAX_DQK) return set_error(XL_ERR_UNSUPPORTED, "%s: DQK %d is over %d", who, s.DK, MAX_DQK);
  if (s.DV > (1 << 20)) return set_error(XL_ERR_UNSUPPORTED, "%s: DV %d is over 2^20", who, s.DV);
  const int64_t heads = (int64_t)s.B * s.NH, chunks = s.chunks() + 1;
  if (heads >= (1 << 24) || heads * chunks * ((s.DV + 15) / 16) >= ((int64_t)1 << 31))
    return set_error(XL_ERR_UNSUPPORTED, "%s: B NH S DV too large", who);
  return XL_OK;
}

int set_strides(Shape& s, const int64_t* strides, const char* who) {
  if (strides) {
    for (int i = 0; i < 3; ++i)  // a token stride is multiplied by up to 63 in 32 bits
      if (strides[3 * i + 2] < 0 || strides[3 * i + 2] > MAX_TOKEN_STRIDE)
        return set_error(XL_ERR_UNSUPPORTED, "%s: token strides must be 0 to %d elements", who, MAX_TOKEN_STRIDE);
    for (int i = 0; i < 3; ++i) {
      s.qs[i] = strides[i];
      s.ks[i] = strides[3 + i];
      s.vs[i] = strides[6 + i];
    }
    return XL_OK;
  }
  auto dense = [&](int64_t (&to)[3], int heads, int D) {
    to[2] = D;
    to[1] = (int64_t)s.S * D;
    to[0] = to[1] * heads;
  };
  dense(s.qs, s.NHK, s.DK);
  dense(s.ks, s.NHK, s.DK);
  dense(s.vs, s.NH, s.DV);
  return XL_OK;
}

int launch_recurrent(const Shape& s, const void* q, const void* k, const void* v, const void* g, const void* beta,
                     const float* c0, void* h, float* c_last, hipStream_t st, const char* who) {
  RecArgs a{q, k, v, g, beta, c0, h, c_last, s.NH, s.NH / s.NHK, s.S, s.DK, s.DV, s.scale, false};
  a.wide = s.DV % 4 == 0 && (((uintptr_t)c0 | (uintptr_t)c_last) & 15) == 0;
  const void* kern = nullptr;
  auto with_gate = [&](auto t) {
    using T = decltype(t);
    kern = s.dtype_gates == XL_DTYPE_F32 ? pick<T, float>(s.DK) : s.dtype_gates == XL_DTYPE_BF16 ? pick<T, bf16_t>(s.DK) : pick<T, f16_t>(s.DK);
  };
  if (s.dtype == XL_DTYPE_F32) with_gate(float{});
  else if (s.dtype == XL_DTYPE_BF16) with_gate(bf16_t{});
  else with_gate(f16_t{});
  const unsigned grid = (unsigned)((int64_t)s.B * s.NH * ((s.DV + COLS - 1) / COLS));
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(kern, dim3(grid), dim3(256), args, 0, st);
  if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
  return check_launch(who);
}

}  // namespace delta
}  // namespace xl

extern "C" int xl_gated_delta_recurrent_fwd(const void* q, const void* k, const void* v, const void* g, const void* beta,
                                            const float* c0, void* h, float* c_last, int B, int NH, int NHK, int S, int DQK,
                                            int DV, float scale, int dtype_qkv, int dtype_gates, void* stream) {
  using namespace xl;
  const char* who = "xl_gated_delta_recurrent_fwd";
  clear_error();
  delta::Shape s{B, NH, NHK, S, DQK, DV, {}, {}, {}, scale, dtype_qkv, dtype_gates};
  if (const int rc = delta::check_shape(who, s)) return rc;
  if (S > 0 && (!q || !k || !v || !g || !beta || !h)) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (S == 0 && !c_last) return XL_OK;
  return delta::launch_recurrent(s, q, k, v, g, beta, c0, h, c_last, (hipStream_t)stream, who);
}
