// Gated delta rule token by token (decode steps, a few drafted tokens):
//
//   S = a S + k d^T,  d = beta (v - a S^T k),  h = scale S^T q,  a = exp(g)
//
// A workgroup takes 32 columns of a head's state through all tokens, in float32 registers: 4 waves x 8 lane groups share
// the rows, a lane holds 4 columns of every 32nd row.  S^T k and S^T q of the state before the token are summed
// together (h = scale (a S^T q + (q.k) d)), so a token costs one reduction and one barrier; the next token's values are on their
// way meanwhile.  13 tokens of 32 heads of 128 x 256 (bf16): 16.9 us, 1 a token, bound by that reduction's latency.  One token
// is bound by the state's bytes, in and out once, and has a kernel of its own.
#include "delta.h"

namespace xl {
namespace delta {
namespace {

constexpr int COLS = 32, RWAVES = 4;
static_assert(MAX_DQK == 64 * RWAVES);  // a thread for each value of q and k

struct RecArgs {
  const void *q, *k, *v, *g, *beta;
  const float* c0;
  void* h;
  float* c_last;
  int NH, group, S, DK, DV;
  float scale;
  bool wide;  // 16-byte accesses to the state
};

// x + what the lanes 8, 16 and 32 away have: the sum over a wave's 8 row groups
__device__ __forceinline__ float sum_groups(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));  // row_ror:8
  const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(y[0]) + __uint_as_float(y[1]);
  const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(z[0]) + __uint_as_float(z[1]);
}

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
  // Thread tid has value tid of a token's q and k.  What is loaded past the last token or value is the last one's.  No branch around a load: the compiler would wait for it at the branch's end.
  const int dc = tid < p.DK ? tid : p.DK - 1;
  T qn{}, kn{};
  auto load_qk = [&](int t) {
    const int64_t at = (int64_t)(t < p.S ? t : p.S - 1) * p.DK + dc;
    qn = q[at];
    kn = k[at];
  };
  if (p.S > 0) {
    load_qk(0);
    qk_s[0][0][tid] = to_f32(qn);
    qk_s[0][1][tid] = to_f32(kn);
    load_qk(1);
  }
  T vn[4];
  G gn{}, bn{};
  int vcol[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) vcol[e] = col + e < p.DV ? col + e : p.DV - 1;
  auto load = [&](int t) {
    t = t < p.S ? t : p.S - 1;
    gn = gp[t];
    bn = bp[t];
#pragma unroll
    for (int e = 0; e < 4; ++e) vn[e] = v[(int64_t)t * p.DV + vcol[e]];
  };
  if (p.S > 0) load(0);
  lds_barrier();
  for (int t = 0; t < p.S; ++t) {
    const int at = t & 1;
    const float a = expf(to_f32(gn)), beta = to_f32(bn);
    float vt[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) vt[e] = to_f32(vn[e]);
    qk_s[at ^ 1][0][tid] = to_f32(qn);  // the next token's, read a token ago
    qk_s[at ^ 1][1][tid] = to_f32(kn);
    load(t + 1);
    load_qk(t + 2);
    f32x4 ks = {0.f, 0.f, 0.f, 0.f}, qs = {0.f, 0.f, 0.f, 0.f};
    float kk[NI], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const bool there = row0 + 32 * i < p.DK;
      const float qi = there ? qk_s[at][0][row0 + 32 * i] : 0.f;
      kk[i] = there ? qk_s[at][1][row0 + 32 * i] : 0.f;
      dot = fmaf(qi, kk[i], dot);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] = fmaf(kk[i], st[i][e], ks[e]);
        qs[e] = fmaf(qi, st[i][e], qs[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ks[e] = sum_groups(ks[e]);
      qs[e] = sum_groups(qs[e]);
    }
    dot = sum_groups(dot);
    if (lane < 8) {
      *(f32x4*)&sums[at][wave][0][lane * 4] = ks;
      *(f32x4*)&sums[at][wave][1][lane * 4] = qs;
      if (lane == 0) dots[at][wave] = dot;
    }
    lds_barrier();
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

// One token: 1024 threads a workgroup, COLS columns (256: a wave reads whole KBs of a row), every thread's rows read
// before the first is written.  S^T k and S^T q are summed over a thread's rows, then over the row groups in LDS.
constexpr int STEP_THREADS = 1024;

template <typename T, typename G, int COLS, int DKP>
__global__ __launch_bounds__(STEP_THREADS) void delta_step_kernel(RecArgs p) {
  constexpr int CG = COLS / 4, RG = STEP_THREADS / CG, RPT = DKP / RG, LANES = STEP_THREADS / COLS;
  static_assert(RG == 4 * LANES && DKP % RG == 0);
  __shared__ float q_s[DKP], k_s[DKP], sums[2][RG][COLS + 4], d_s[COLS], dots[STEP_THREADS / 64];
  const int tid = threadIdx.x, tiles = (p.DV + COLS - 1) / COLS;
  const int bh = uniform(blockIdx.x / tiles), tile = blockIdx.x - bh * tiles, b = uniform(bh / p.NH), h = bh - b * p.NH;
  const int64_t bhk = (int64_t)b * uniform(p.NH / p.group) + uniform(h / p.group);
  const int cg = tid % CG, rg = tid / CG, col = tile * COLS + cg * 4, colc = col < p.DV ? col : 0;
  // the small values first, then the rows (past DQK: row 0 again, against zeros), all under way at once
  const G graw = ((const G*)p.g)[bh], braw = ((const G*)p.beta)[bh];
  const int d0 = tid < p.DK ? tid : 0;
  const T qraw = ((const T*)p.q)[bhk * p.DK + d0], kraw = ((const T*)p.k)[bhk * p.DK + d0];
  const int own = tile * COLS + tid / LANES;  // the column that this thread helps to sum
  const T vraw = ((const T*)p.v)[(int64_t)bh * p.DV + (own < p.DV ? own : 0)];
  asm volatile("" ::: "memory");
  const int64_t state = (int64_t)bh * p.DK * p.DV + colc;
  f32x4 st[RPT];
  if (p.wide) {
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = rg + RG * i;
      st[i] = __builtin_nontemporal_load((const f32x4*)(p.c0 + state + (int64_t)(r < p.DK ? r : 0) * p.DV));
    }
  } else {  // columns past the last: that one again
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = rg + RG * i;
      const float* from = p.c0 + state + (int64_t)(r < p.DK ? r : 0) * p.DV;
#pragma unroll
      for (int e = 0; e < 4; ++e) st[i][e] = from[colc + e < p.DV ? e : p.DV - 1 - colc];
    }
  }
  const float qv = tid < p.DK ? to_f32(qraw) : 0.f, kv = tid < p.DK ? to_f32(kraw) : 0.f;
  if (tid < DKP) {
    q_s[tid] = qv;
    k_s[tid] = kv;
  }
  const float part = wave_sum(qv * kv);
  if ((tid & 63) == 0) dots[tid >> 6] = part;
  const float a = expf(to_f32(graw)), beta = to_f32(braw);
  lds_barrier();
  float kk[RPT];
  f32x4 ks = {0.f, 0.f, 0.f, 0.f}, qs = ks;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    kk[i] = k_s[rg + RG * i];
    const float qi = q_s[rg + RG * i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ks[e] = fmaf(kk[i], st[i][e], ks[e]);
      qs[e] = fmaf(qi, st[i][e], qs[e]);
    }
  }
  *(f32x4*)&sums[0][rg][cg * 4] = ks;
  *(f32x4*)&sums[1][rg][cg * 4] = qs;
  lds_barrier();
  {
    const int c = tid / LANES, l = tid % LANES;
    float x[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      x[m] = (sums[m][l][c] + sums[m][l + LANES][c]) + (sums[m][l + 2 * LANES][c] + sums[m][l + 3 * LANES][c]);
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) x[m] += __shfl_xor(x[m], o, 64);
    }
    if (l == 0 && own < p.DV) {
      float dot = 0.f;
#pragma unroll
      for (int w = 0; w < (DKP + 63) / 64; ++w) dot += dots[w];
      const float d = beta * (to_f32(vraw) - a * x[0]);
      d_s[c] = d;
      ((T*)p.h)[(int64_t)bh * p.DV + own] = from_f32<T>(p.scale * fmaf(dot, d, a * x[1]));
    }
  }
  lds_barrier();
  if (col >= p.DV || !p.c_last) return;
  const f32x4 d = *(const f32x4*)&d_s[cg * 4];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg + RG * i;
    if (r >= p.DK) continue;
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaf(kk[i], d[e], a * st[i][e]);
    float* const to = p.c_last + state + (int64_t)r * p.DV;
    if (p.wide) {
      __builtin_nontemporal_store(x, (f32x4*)to);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.DV) to[e] = x[e];
    }
  }
}

template <typename T, typename G, int COLS>
const void* pick_step(int DK) {
  if constexpr (COLS == 64)
    return DK <= 64 ? (const void*)delta_step_kernel<T, G, COLS, 64> : DK <= 128 ? (const void*)delta_step_kernel<T, G, COLS, 128>
                                                                                : (const void*)delta_step_kernel<T, G, COLS, 256>;
  return DK <= 128 ? (const void*)delta_step_kernel<T, G, 256, 128> : (const void*)delta_step_kernel<T, G, 256, 256>;
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
  // One token from a state: 1 KB rows where that gives every CU a workgroup, else 256-byte ones, else the kernel of
  // several tokens.  bf16, us, in that order: 8 heads of 128 x 256 6.1, 4.3, 5.3; 64 heads 6.7, 5.7, 7.5; 256 heads 12.4, 14.9, 17.6;
  // 16 heads of 256 x 512 9.6, 6.0, 10.4; 128 heads 23.9, 26.8, 41.0 (268 MB: 5.6 TB/s).
  const int64_t heads = (int64_t)s.B * s.NH;
  const bool one = s.S == 1 && c0;
  const int cols = !one ? 0 : s.DV % 256 == 0 && heads * (s.DV / 256) >= 256 ? 256 : 64;
  const void* kern = nullptr;
  auto with_gate = [&](auto t) {
    using T = decltype(t);
    auto of = [&](auto g) {
      using G = decltype(g);
      kern = cols == 256 ? pick_step<T, G, 256>(s.DK) : cols == 64 ? pick_step<T, G, 64>(s.DK) : pick<T, G>(s.DK);
    };
    if (s.dtype_gates == XL_DTYPE_F32) of(float{});
    else if (s.dtype_gates == XL_DTYPE_BF16) of(bf16_t{});
    else of(f16_t{});
  };
  if (s.dtype == XL_DTYPE_F32) with_gate(float{});
  else if (s.dtype == XL_DTYPE_BF16) with_gate(bf16_t{});
  else with_gate(f16_t{});
  const int width = cols ? cols : COLS;
  const unsigned grid = (unsigned)(heads * ((s.DV + width - 1) / width));
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(kern, dim3(grid), dim3(cols ? STEP_THREADS : 256), args, 0, st);
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
