// Gated delta rule token by token (decode steps, a few drafted tokens):
//
//   S = a S + k d^T,  d = beta (v - a S^T k),  h = scale S^T q,  a = exp(g)
//
// A workgroup takes 32 or 16 columns of a head's state through all tokens, in float32 registers: 4 waves x 8 or 16 lane
// groups share the rows, a lane holds 4 columns of every 32nd or 64th row.  S^T k and S^T q of the state before the token are
// summed together (h = scale (a S^T q + (q.k) d)), so a token costs one reduction and one barrier, whose latency bounds it:
// 13 tokens of 32 heads of 128 x 256 (bf16) 11.0 us, 0.6 a token.  Tokens' values come 8 tokens at a time and a block ahead.
// One token is bound by the state's bytes, in and out once, and has a kernel of its own.
#include "delta.h"

namespace xl {
namespace delta {
namespace {

constexpr int RWAVES = 4;

struct RecArgs {
  const void *q, *k, *v, *g, *beta;
  const float* c0;
  void* h;
  float* c_last;
  int NH, group, S, DK, DV;
  float scale;
  bool wide;    // 16-byte accesses to the state
  bool wide_h;  // 4 values of h at once
};

// x + what the lanes G, 2 G .. 32 away have: the sum over a wave's lane groups
template <int G>
__device__ __forceinline__ float sum_row(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));  // row_ror:8
  if (G == 4) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xf, 0xf, false));  // row_ror:4
  return x;
}
// both sums over halves of the wave: a's in its lower half (of 32 or, alternately, of 16 lanes), b's in the upper
__device__ __forceinline__ float fold32(float a, float b) {
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {
  const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

template <typename T, typename G, int COLS, int DKP>
__global__ __launch_bounds__(256) void delta_recurrent_kernel(RecArgs p) {
  constexpr int QUADS = COLS / 4, RSTEP = RWAVES * 64 / QUADS, NI = DKP / RSTEP;
  static_assert(NI * RSTEP == DKP);
  // a block of tokens' values, brought by one load a thread for each of PASSES tokens of q and k, for v, g and beta
  constexpr int TOKENS = 8, AT_ONCE = 256 / DKP, PASSES = TOKENS / AT_ONCE;
  __shared__ float q_s[TOKENS][DKP], k_s[TOKENS][DKP], v_s[TOKENS][COLS], gates[TOKENS][2];
  __shared__ float sums[2][RWAVES][2][COLS];
  __shared__ float dots[2][RWAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lg = lane / QUADS, quad = lane % QUADS;
  const int slices = (p.DV + COLS - 1) / COLS;
  const int all = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int bh = all / slices, col = (all - bh * slices) * COLS + quad * 4;
  const int b = bh / p.NH, h = bh - b * p.NH, bhk = b * (p.NH / p.group) + h / p.group;
  const T* q = (const T*)p.q + (int64_t)bhk * p.S * p.DK;
  const T* k = (const T*)p.k + (int64_t)bhk * p.S * p.DK;
  const T* v = (const T*)p.v + (int64_t)bh * p.S * p.DV;
  T* ho = (T*)p.h + (int64_t)bh * p.S * p.DV;
  const G *gp = (const G*)p.g + (int64_t)bh * p.S, *bp = (const G*)p.beta + (int64_t)bh * p.S;
  const int64_t state = (int64_t)bh * p.DK * p.DV;
  const int row0 = wave * (64 / QUADS) + lg;

  // Rows past DQK are the first again, against zeros, and columns past DV the last.
  f32x4 st[NI];
  const int colc = min(col, p.DV - 1);
  if (p.c0 && p.wide) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = row0 + RSTEP * i;
      st[i] = __builtin_nontemporal_load((const f32x4*)(p.c0 + state + (int64_t)(r < p.DK ? r : 0) * p.DV + (col < p.DV ? col : 0)));
    }
  } else if (p.c0) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = row0 + RSTEP * i;
      const float* from = p.c0 + state + (int64_t)(r < p.DK ? r : 0) * p.DV;
#pragma unroll
      for (int e = 0; e < 4; ++e) st[i][e] = from[min(colc + e, p.DV - 1)];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i) st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // What is loaded past the last token or column is the last one's, past the last value a zero.  No branch around a load: the
  // compiler would wait for it at the branch's end.
  T qn[PASSES], kn[PASSES], vn{};
  G gn{}, bn{};
  const int value = tid % DKP, vtoken = tid / COLS, vcol = (all - bh * slices) * COLS + tid % COLS;
  const bool there = value < p.DK;
  auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int64_t at = (int64_t)min(t0 + i * AT_ONCE + tid / DKP, p.S - 1) * p.DK + (there ? value : 0);
      qn[i] = q[at];
      kn[i] = k[at];
    }
    vn = v[(int64_t)min(t0 + vtoken, p.S - 1) * p.DV + min(vcol, p.DV - 1)];
    const int t = min(t0 + (tid & (TOKENS - 1)), p.S - 1);
    gn = gp[t];
    bn = bp[t];
  };
  if (p.S > 0) load(0);
  // here, not at its first use: in the loop that wait would be for every token's stores too
#pragma unroll
  for (int i = 0; i < NI; ++i) asm volatile("" : "+v"(st[i]));
  for (int t = 0; t < p.S; ++t) {
    const int at = t & 1, in = t & (TOKENS - 1);
    if (in == 0) {  // the block before has been read: each token's values before its barrier
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        q_s[i * AT_ONCE + tid / DKP][value] = there ? to_f32(qn[i]) : 0.f;
        k_s[i * AT_ONCE + tid / DKP][value] = there ? to_f32(kn[i]) : 0.f;
      }
      if (vtoken < TOKENS) v_s[vtoken][tid % COLS] = to_f32(vn);
      if (tid < TOKENS) {
        gates[tid][0] = expf(to_f32(gn));
        gates[tid][1] = to_f32(bn);
      }
      load(t + TOKENS);
      lds_barrier();
    }
    const float a = gates[in][0], beta = gates[in][1];
    const f32x4 vt = *(const f32x4*)&v_s[in][quad * 4];
    f32x4 ks = {0.f, 0.f, 0.f, 0.f}, qs = {0.f, 0.f, 0.f, 0.f};
    float kk[NI], dot = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float qi = q_s[in][row0 + RSTEP * i];
      kk[i] = k_s[in][row0 + RSTEP * i];
      dot = fmaf(qi, kk[i], dot);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] = fmaf(kk[i], st[i][e], ks[e]);
        qs[e] = fmaf(qi, st[i][e], qs[e]);
      }
    }
    // lanes below 32 get the sums of S^T k, the others S^T q's; of those, 16 lanes the columns 0 and 2, 16 the columns 1 and 3
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = fold32(ks[e], qs[e]);
    const float s02[2] = {sum_row<QUADS>(fold16(y[0], y[1])), sum_row<QUADS>(fold16(y[2], y[3]))};
    dot = fold32(dot, dot);
    dot = sum_row<QUADS>(fold16(dot, dot));
    if ((lane & 15) < QUADS) {
      float* to = &sums[at][wave][lane >> 5][quad * 4 + (lane >> 4 & 1)];
      to[0] = s02[0];
      to[2] = s02[1];
    }
    if (lane == 0) dots[at][wave] = dot;
    lds_barrier();
    f32x4 part[RWAVES];
#pragma unroll
    for (int w = 0; w < RWAVES; ++w) part[w] = *(const f32x4*)&sums[at][w][0][quad * 4];
    __builtin_amdgcn_sched_barrier(0);  // all four under way at once
    ks = (part[0] + part[1]) + (part[2] + part[3]);
    f32x4 d;
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = beta * (vt[e] - a * ks[e]);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) st[i][e] = fmaf(kk[i], d[e], a * st[i][e]);
    if (wave == (t & (RWAVES - 1)) && lg == 0) {  // the waves in turn
      dot = 0.f;
#pragma unroll
      for (int w = 0; w < RWAVES; ++w) {
        part[w] = *(const f32x4*)&sums[at][w][1][quad * 4];
        dot += dots[at][w];
      }
      qs = (part[0] + part[1]) + (part[2] + part[3]);
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = p.scale * fmaf(dot, d[e], a * qs[e]);
      const Four<T> o = rounded4<T>(y);
      T* const to = ho + (int64_t)t * p.DV + col;
      if (p.wide_h) {
        if (col < p.DV) *(Four<T>*)to = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.DV) to[e] = o.e[e];
      }
    }
  }
  if (!p.c_last) return;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = row0 + RSTEP * i;
    if (r >= p.DK) continue;
    float* to = p.c_last + state + (int64_t)r * p.DV + col;
    if (p.wide) {
      if (col < p.DV) *(f32x4*)to = st[i];
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

template <typename T, typename G, int COLS>
const void* pick(int DK) {
  return DK <= 64 ? (const void*)delta_recurrent_kernel<T, G, COLS, 64> : DK <= 128 ? (const void*)delta_recurrent_kernel<T, G, COLS, 128>
                                                                                 : (const void*)delta_recurrent_kernel<T, G, COLS, 256>;
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
  // a launch has fewer than 2^32 threads: 256 for 32 columns of a head
  if (heads * ((s.DV + 31) / 32) >= (1 << 24)) return set_error(XL_ERR_UNSUPPORTED, "%s: B NH DV too large", who);
  return XL_OK;
}

int set_strides(Shape& s, const int64_t* strides, const char* who) {
  if (strides) {
    for (int i = 0; i < 3; ++i)  // a token stride is multiplied by up to 63 in 32 bits; one token's is never stepped
      if (s.S > 1 && (strides[3 * i + 2] < 0 || strides[3 * i + 2] > MAX_TOKEN_STRIDE))
        return set_error(XL_ERR_UNSUPPORTED, "%s: token strides must be 0 to %d elements", who, MAX_TOKEN_STRIDE);
    for (int i = 0; i < 3; ++i) {
      s.qs[i] = strides[i];
      s.ks[i] = strides[3 + i];
      s.vs[i] = strides[6 + i];
    }
    if (s.S <= 1) s.qs[2] = s.ks[2] = s.vs[2] = 0;
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
  RecArgs a{q, k, v, g, beta, c0, h, c_last, s.NH, s.NH / s.NHK, s.S, s.DK, s.DV, s.scale, false, false};
  a.wide_h = s.DV % 4 == 0 && (uintptr_t)h % 16 == 0;
  a.wide = s.DV % 4 == 0 && (((uintptr_t)c0 | (uintptr_t)c_last) & 15) == 0;
  // One token from a state: 1 KB rows where that gives every CU a workgroup, else 256-byte ones, else the kernel of
  // several tokens.  bf16, us, in that order: 8 heads of 128 x 256 6.1, 4.3, 5.3; 64 heads 6.7, 5.7, 7.5; 256 heads 12.4, 14.9, 17.6;
  // 16 heads of 256 x 512 9.6, 6.0, 10.4; 128 heads 23.9, 26.8, 41.0 (268 MB: 5.6 TB/s).
  const int64_t heads = (int64_t)s.B * s.NH;
  const bool one = s.S == 1 && c0 && heads * ((s.DV + 63) / 64) < (1 << 22);  // 2^32 threads
  const int step = !one ? 0 : s.DV % 256 == 0 && heads * (s.DV / 256) >= 256 ? 256 : 64;
  // Several: 16 columns a workgroup where 32 give a CU one at most, for 13 tokens of 128 x 256 us of 16 and 32: 8 heads 10.2, 11.3; 32
  // heads 12.2, 12.5; 64 heads 17.5, 14.8; 128 heads 28.9, 21.4.
  const int width = step ? step : heads * ((s.DV + 31) / 32) <= 256 ? 16 : 32;
  const void* kern = nullptr;
  auto with_gate = [&](auto t) {
    using T = decltype(t);
    auto of = [&](auto g) {
      using G = decltype(g);
      kern = step == 256 ? pick_step<T, G, 256>(s.DK)
             : step == 64 ? pick_step<T, G, 64>(s.DK)
             : width == 16 ? pick<T, G, 16>(s.DK)
                           : pick<T, G, 32>(s.DK);
    };
    if (s.dtype_gates == XL_DTYPE_F32) of(float{});
    else if (s.dtype_gates == XL_DTYPE_BF16) of(bf16_t{});
    else of(f16_t{});
  };
  if (s.dtype == XL_DTYPE_F32) with_gate(float{});
  else if (s.dtype == XL_DTYPE_BF16) with_gate(bf16_t{});
  else with_gate(f16_t{});
  const unsigned grid = (unsigned)(heads * ((s.DV + width - 1) / width));
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(kern, dim3(grid), dim3(step ? STEP_THREADS : 256), args, 0, st);
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
