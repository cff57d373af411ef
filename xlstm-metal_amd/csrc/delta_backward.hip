// Gradients of the gated delta rule by chunks (delta.h has the forward's formulas).  From dH and dS, the gradient of the state
// behind a chunk:
//
//   dU = P^T dH + diag(c_L / c_j) K dS,  Z = T^T dU,  dV = diag(beta) Z,
//   dS_0 = c_L dS + scale (diag(c) Q)^T dH - (diag(c beta) K)^T Z
//
// are again of each column by itself: a scan from the last chunk to the first, built as the forward's.  U and the states
// are formed again by the forward's scan.  Both scans keep U, Z, S_0 and dS in f16 planes for the last kernel, a workgroup a
// chunk, which sums over the columns:
//
//   dP = dH U^T (j <= i),  dA = -Z U^T (j < i),  N_ij = D_ij k_i.k_j,  E_ij = dA_ij beta_i D_ij
//   dQ = scale (diag(c) dH S_0^T + (D o dP) K)
//   dK = diag(c_L / c_j) U dS^T - diag(c beta) Z S_0^T + scale (D o dP)^T Q + (E + E^T) K
//   dbeta_i = Z_i.V_i - c_i k_i.(Z S_0^T)_i + sum_j dA_ij N_ij
//
// and for dg every term's exponent b_i - b_j, which b_i gets and b_j loses: rows and columns of dP o P and dA o A, q.dQ's and
// k.dK's parts with the states, c_L <dS, S_0>; dg_t is the sum of b's gradients from t to the chunk's end.  (The same numbers
// are added at a term's later token and taken off at its earlier one, so what does not pass t cancels to float32's rounding.)
//
// Heads of v that share q and k write their dQ and dK in float32, and a last kernel adds them in order.
//
// Measured (2 x 4096 tokens of 8 heads of 128 x 256), us: first kernel 37, dH by columns 17, states 124, scan backwards 163, chunks'
// gradients 134 for bf16 inputs and gates; with float32 gates, which keep pairs, 37, 22, 149, 189, 270.  The scans are bound by the chain of one chunk's step; the last by its waits between products
// (its 377 MB are 73 us of a copy).
#include "delta.h"

namespace xl {
namespace delta {
namespace {

// ------------------------------------------------------------------------------------------------ dH by columns
struct TurnArgs {
  const void* dh;
  Kept kept;
  int S, DV, chunks;
  bool wide;  // 16-byte loads
};

template <typename T, int KEPT>
__global__ __launch_bounds__(256) void delta_turn_kernel(TurnArgs p) {
  __shared__ float tile[L][65];
  const int64_t part = blockIdx.x;
  const int64_t bh = part / p.chunks;
  const int t0 = (int)(part - bh * p.chunks) * L, n0 = blockIdx.y * 64;
  // 8 lanes a row, 8 values each
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = half * 32 + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 8;
    const T* from = (const T*)p.dh + (bh * p.S + t0 + row) * p.DV + n0 + c;
    float x[8];
    if (t0 + row < p.S && n0 + c + 8 <= p.DV && p.wide) {
      struct alignas(16) Eight { T e[8]; };
      const Eight v = *(const Eight*)from;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = to_f32(v.e[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = t0 + row < p.S && n0 + c + e < p.DV ? to_f32(from[e]) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[row][c + e] = x[e];
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, gq = lane >> 4, block = blockIdx.y * 4 + wave;
  if (block >= p.kept.blocks) return;
  float x[2][8], m = 0.f;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[s][e] = tile[32 * s + (e < 4 ? 4 * gq + e : 12 + 4 * gq + e)][16 * wave + r];
      m = fmaxf(m, fabsf(x[s][e]));
    }
  const Pow2 sc = pow2_for(wave_max_all(m));
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    f16x8 hi, lo;
    split8<KEPT == 2>(x[s], sc.up, hi, lo);
    f16_t* to = p.kept.dh + kept_at(part, p.kept.blocks, block, KEPT, L) + r * L + s * 32 + gq * 8;
    *(f16x8*)to = hi;
    if constexpr (KEPT == 2) *(f16x8*)(to + 16 * L) = lo;
  }
  if (lane == 0) p.kept.dhs[part * p.kept.blocks + block] = sc.down;
}

// ------------------------------------------------------------------------------------------------ the scan backwards
struct BackArgs {
  const float* dc_last;
  float* dc0;
  Prep prep;
  Kept kept;
  int NH, group, DK, DV, chunks, slices;
};

// As the forward's scan (delta_chunkwise.hip): operands are read ahead of their products, the next chunk's are on their way.
// Four waves take a block each and bring the images together; a wave on its own has a second one that only brings them (a load into
// LDS that has to queue stops its wave: 177 us without, 157 with, at 8192 tokens of 128 x 256, 2.5 a chunk).
template <typename T, int DKB, int STAGES, int W, int KEPT>
__global__ __launch_bounds__(W == 1 ? 128 : 64 * W, 1) void delta_back_kernel(BackArgs p) {
  constexpr int DKP = DKB * 32, PK = PLANES<T>, PLANE = L * DKP * 2, IMG = PK * PLANE, STAGE = 2 * IMG;
  extern __shared__ __align__(1024) char lds[];  // STAGES of K and Q; two chunks' factors
  const int lane = threadIdx.x & 63, in = uniform(threadIdx.x >> 6), wave = W == 1 ? 0 : in;
  const int r = lane & 15, gq = lane >> 4;
  const int all = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int bh = uniform(all / p.slices), slice = all - bh * p.slices, b = uniform(bh / p.NH), h = bh - b * p.NH;
  const int64_t image0 = ((int64_t)b * uniform(p.NH / p.group) + uniform(h / p.group)) * p.chunks, part0 = (int64_t)bh * p.chunks;
  // past the last block a wave computes it again and writes nothing
  const int own = slice * W + wave, block = own < p.kept.blocks ? own : p.kept.blocks - 1, n = block * 16 + r;
  const bool mine = own < p.kept.blocks;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_char*)lds;
  // a chunk's images, in DKB shares; a wave brings every W-th KB
  constexpr int SHARE = STAGE / 1024 / DKB / W;
  static_assert(SHARE * W * DKB * 1024 == STAGE);
  auto fetch = [&](int chunk, int stage, int share) {
    const char* ki = p.prep.k + (image0 + chunk) * (int64_t)IMG;
    const char* qi = p.prep.q + (image0 + chunk) * (int64_t)IMG - IMG;
#pragma unroll
    for (int j = 0; j < SHARE; ++j) {
      const int i = (share * SHARE + j) * W;  // K's or Q's, for all waves
      to_lds(lds_at + stage * STAGE + (i + wave) * 1024, (i + wave) * 1024 + lane * 16, i < IMG / 1024 ? ki : qi);
    }
  };
  auto fetch_factors = [&](int chunk) {
    if (wave != 0) return;
    to_lds(lds_at + STAGES * STAGE + (chunk & 1) * 2048, lane * 16, p.prep.f + part0 + chunk);
    to_lds(lds_at + STAGES * STAGE + (chunk & 1) * 2048 + 1024, 1024 + lane * 16, p.prep.f + part0 + chunk);
  };
  const int last = p.chunks - 1;
  if (W == 1 && in == 1) {
    for (int c = last; c >= 0; --c) {  // the other wave's barriers
      if (c == last || STAGES == 1) {
#pragma unroll
        for (int s = 0; s < DKB; ++s) fetch(c, STAGES == 2 ? c & 1 : 0, s);
        fetch_factors(c);
      }
      wait_loads();
      lds_barrier();
      if (STAGES == 2 && c > 0) {
#pragma unroll
        for (int s = 0; s < DKB; ++s) fetch(c - 1, (c - 1) & 1, s);
        fetch_factors(c - 1);
      }
      if (STAGES == 1) lds_barrier();
    }
    return;
  }
  f32x4 st[2 * DKB];  // the state's gradient times 1 / st_down
#pragma unroll
  for (int t = 0; t < 2 * DKB; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * t + 4 * gq + e;
      st[t][e] = p.dc_last && d < p.DK && n < p.DV ? p.dc_last[((int64_t)bh * p.DK + d) * p.DV + n] : 0.f;
    }
  float st_down;
  {
    const Pow2 sc = pow2_for(state_max(st), STATE_BACK);
    st_down = sc.down;
#pragma unroll
    for (int t = 0; t < 2 * DKB; ++t) st[t] *= sc.up;
  }
  f16x8 th[LOWER], tl[LOWER], ph[LOWER], pl[LOWER], dh[2], dl[2];
  float dh_scale = 0.f;
  auto load_t = [&](int chunk) {
    const f16_t* from = p.prep.tt + (part0 + chunk) * (2 * FRAG_PLANE);
    load_upper(from, lane, th);
    load_upper(from + FRAG_PLANE, lane, tl);
  };
  auto load_p = [&](int chunk) {
    const f16_t* from = p.prep.pt + (part0 + chunk) * (2 * FRAG_PLANE);
    load_upper(from, lane, ph);
    load_upper(from + FRAG_PLANE, lane, pl);
  };
  auto load_dh = [&](int chunk) {
    const f16_t* from = p.kept.dh + kept_at(part0 + chunk, p.kept.blocks, block, KEPT, L);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      dh[s] = load16(from, r * (L * 2) + gq * 16 + s * 64);
      if constexpr (KEPT == 2) dl[s] = load16(from + 16 * L, r * (L * 2) + gq * 16 + s * 64);
    }
    dh_scale = p.kept.dhs[(part0 + chunk) * p.kept.blocks + block];
  };
  if (W != 1) {
#pragma unroll
    for (int s = 0; s < DKB; ++s) fetch(last, STAGES == 2 ? last & 1 : 0, s);
    fetch_factors(last);
  }
  load_p(last);
  load_t(last);
  load_dh(last);
  for (int c = last; c >= 0; --c) {
    // The chunk's only wait for memory.  The compiler does not count the loads into LDS: a wait of its own for a register,
    // behind them, would be for all of them too, and they have only just left.
    wait_loads();
    lds_barrier();
    const int stage = STAGES == 2 ? c & 1 : 0, next = c > 0 ? c - 1 : c;
    if (W != 1 && next != c) fetch_factors(next);
    const char *ki = lds + stage * STAGE, *qi = ki + IMG;
    const Factors* f = (const Factors*)(lds + STAGES * STAGE + (c & 1) * 2048);
    const int64_t at = (part0 + c) * p.kept.blocks + block;
    // ---- K dS; dS is kept
    f16x8 rows[2][PK][4];
    auto read = [&](int s) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int pl = 0; pl < PK; ++pl) rows[s & 1][pl][mt] = rows_frag<DKP>(ki + pl * PLANE, mt, s, r, gq);
    };
    read(0);
    f32x4 ks[4], out[4], fq[4], fb[4], fp[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      ks[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      out[mt] = *(const f32x4*)&f->out[16 * mt + 4 * gq] * st_down;
      fq[mt] = *(const f32x4*)&f->q[16 * mt + 4 * gq];
      fb[mt] = *(const f32x4*)&f->back[16 * mt + 4 * gq];
      fp[mt] = *(const f32x4*)&f->pt[16 * mt + 4 * gq] * dh_scale;
    }
    const float keep = f->all, t_scale = f->tt;
    f16_t* const to_ds = p.kept.ds + kept_at(part0 + c, p.kept.blocks, block, KEPT, DKP);
    f16x8 sh[2], sl[2];
    split8(st[0], st[1], sh[0], sl[0]);
#pragma unroll
    for (int s = 0; s < DKB; ++s) {
      if (s + 1 < DKB) read(s + 1);
      if (W != 1 && STAGES == 2) fetch(next, stage ^ 1, s);
      __builtin_amdgcn_sched_barrier(0);
      const f16x8 hi = sh[s & 1], lo = sl[s & 1];
      if (mine) {
        *(f16x8*)((char*)to_ds + r * (DKP * 2) + gq * 16 + s * 64) = hi;
        if constexpr (KEPT == 2) *(f16x8*)((char*)(to_ds + 16 * DKP) + r * (DKP * 2) + gq * 16 + s * 64) = lo;
      }
      if (s + 1 < DKB) split8(st[2 * s + 2], st[2 * s + 3], sh[(s + 1) & 1], sl[(s + 1) & 1]);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if constexpr (PK == 2) ks[mt] = mfma(rows[s & 1][1][mt], hi, ks[mt]);
        ks[mt] = mfma(rows[s & 1][0][mt], hi, ks[mt]);
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) ks[mt] = mfma(rows[s & 1][0][mt], lo, ks[mt]);
      interleave<8 + (PK == 2 ? 4 : 0)>();
      __builtin_amdgcn_sched_barrier(0);
    }
    // ---- dU
    f32x4 x[4], du[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) x[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < LOWER; ++i) x[upper_mt(i)] = mfma(ph[i], dh[upper_s(i)], x[upper_mt(i)]);
#pragma unroll
    for (int i = 0; i < LOWER; ++i) x[upper_mt(i)] = mfma(pl[i], dh[upper_s(i)], x[upper_mt(i)]);
    if constexpr (KEPT == 2) {
#pragma unroll
      for (int i = 0; i < LOWER; ++i) x[upper_mt(i)] = mfma(ph[i], dl[upper_s(i)], x[upper_mt(i)]);
    }
    load_p(next);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) du[mt][e] = fmaf(x[mt][e], fp[mt][e], out[mt][e] * ks[mt][e]);
    const Pow2 us = pow2_for(wave_max_all(abs_max(du)));
    f16x8 uh[2], ul[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) split8<true>(du[2 * s], du[2 * s + 1], us.up, uh[s], ul[s]);
    // ---- Z
    f32x4 z[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) z[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < LOWER; ++i) z[upper_mt(i)] = mfma(th[i], uh[upper_s(i)], z[upper_mt(i)]);
#pragma unroll
    for (int i = 0; i < LOWER; ++i) z[upper_mt(i)] = mfma(tl[i], uh[upper_s(i)], z[upper_mt(i)]);
#pragma unroll
    for (int i = 0; i < LOWER; ++i) z[upper_mt(i)] = mfma(th[i], ul[upper_s(i)], z[upper_mt(i)]);
    load_t(next);
    // what does not wait for Z: w1, the state's size, the first operands of the state's products
    f32x4 w1[4], w2[4];
    const float most = state_max(st) * st_down;
    constexpr int AHEAD = PK == 2 ? 2 : 4;
    f16x8 kc[AHEAD][PK][2], qc[AHEAD][PK][2];
    auto read_columns = [&](int t) {
#pragma unroll
      for (int pl = 0; pl < PK; ++pl)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          kc[t % AHEAD][pl][s] = columns_frag<DKP>(ki + pl * PLANE, t, s, r, gq);
          qc[t % AHEAD][pl][s] = columns_frag<DKP>(qi + pl * PLANE, t, s, r, gq);
        }
    };
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) read_columns(t);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float d = (float)dh[mt >> 1][(mt & 1) * 4 + e];
        if constexpr (KEPT == 2) d += (float)dl[mt >> 1][(mt & 1) * 4 + e];
        w1[mt][e] = fq[mt][e] * (d * dh_scale);
      }
    load_dh(next);
    const float back = t_scale * us.down;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      z[mt] *= back;
      w2[mt] = -fb[mt] * z[mt];
    }
    const Pow2 zs = pow2_for(wave_max_all(abs_max(z)));
    const Pow2 ws = pow2_for(fmaxf(wave_max_all(fmaxf(abs_max(w1), abs_max(w2))), most * keep), STATE_BACK);
    f16x8 w1h[2], w1l[2], w2h[2], w2l[2], zh[2], zl[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      split8<true>(w1[2 * s], w1[2 * s + 1], ws.up, w1h[s], w1l[s]);
      split8<true>(w2[2 * s], w2[2 * s + 1], ws.up, w2h[s], w2l[s]);
      split8<KEPT == 2>(z[2 * s], z[2 * s + 1], zs.up, zh[s], zl[s]);
    }
    if (mine) {
      f16_t* to = p.kept.z + kept_at(part0 + c, p.kept.blocks, block, KEPT, L);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        *(f16x8*)((char*)to + r * (L * 2) + gq * 16 + s * 64) = zh[s];
        if constexpr (KEPT == 2) *(f16x8*)((char*)(to + 16 * L) + r * (L * 2) + gq * 16 + s * 64) = zl[s];
      }
      if (lane == 0) {
        p.kept.zs[at] = zs.down;
        p.kept.dss[at] = st_down;
      }
    }
    // ---- dS: Q^T w1 + K^T w2
    const float up = keep * st_down * ws.up;
    st_down = ws.down;
#pragma unroll
    for (int t = 0; t < 2 * DKB; ++t) {
      f32x4 y = {0.f, 0.f, 0.f, 0.f}, y2 = y;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if constexpr (PK == 2) {
          y = mfma(qc[t % AHEAD][1][s], w1h[s], y);
          y2 = mfma(kc[t % AHEAD][1][s], w2h[s], y2);
        }
        y = mfma(qc[t % AHEAD][0][s], w1l[s], y);
        y2 = mfma(kc[t % AHEAD][0][s], w2l[s], y2);
        y = mfma(qc[t % AHEAD][0][s], w1h[s], y);
        y2 = mfma(kc[t % AHEAD][0][s], w2h[s], y2);
      }
      st[t] = fma4(st[t], up, y + y2);
      if (t + AHEAD < 2 * DKB) read_columns(t + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (STAGES == 1) {
      lds_barrier();
      if (W != 1 && next != c) {
#pragma unroll
        for (int s = 0; s < DKB; ++s) fetch(next, 0, s);
      }
    }
  }
  wait_loads();
  if (p.dc0 && mine && n < p.DV) {
#pragma unroll
    for (int t = 0; t < 2 * DKB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 16 * t + 4 * gq + e;
        if (d < p.DK) p.dc0[((int64_t)bh * p.DK + d) * p.DV + n] = st[t][e] * st_down;
      }
  }
}

// ------------------------------------------------------------------------------------------------ a chunk's gradients
struct GradArgs {
  const void* v;
  int64_t vs[3];
  void *dq, *dk, *dv, *dg, *dbeta;  // dq, dk: [B, NHK, S, DK], or float32 [B, NH, S, DK] where heads share
  Prep prep;
  Kept kept;
  int NH, group, S, DK, DV, chunks, gate_dtype;
  float scale;
  bool wide_v;
};

constexpr int GLD = 65;

template <typename T, int DKB, int KEPT>
struct GradLds {
  static constexpr int DKP = DKB * 32;
  static constexpr int TOK = 32 * L * 2, STA = 32 * DKP * 2;  // 32 columns of one plane
  static constexpr int STAGE = KEPT * (3 * TOK + 2 * STA), IMAGE = PLANES<T> * L * DKP * 2;
  static constexpr int KK = L * GLD * 4;
  static constexpr int A = STAGE > IMAGE + KK ? STAGE : IMAGE + KK;  // the columns; then K or Q, and K K^T
  static constexpr int OPERANDS = (std::is_same_v<T, bf16_t> ? 3 : 6) * L * L * 2;
  static constexpr int B = 2 * KK > OPERANDS ? 2 * KK : OPERANDS;  // dP, dA; then their operands
  static constexpr int SMALL = (4 * DKB + 1) * L * 4 + 64 * 4 + L * 8 + 4 * L * 4;
  static constexpr int BYTES = A + B + SMALL;
};

// DKB waves: a wave has 32 of DQK's columns of dQ and dK, turned (columns down, tokens across), and its share of the 64 x 64 tiles.
// At DQK 128 two workgroups fit a CU with 256 registers a lane (bf16: 165 us against 187, measured before it came to 135; pairs would spill).
// bf16's dQ and dK take D o dP and E in one plane, whose rounding is an eighth of their own.
template <typename T, int DKB, int KEPT>
__global__ __launch_bounds__(64 * DKB, (DKB == 4 && KEPT == 1 ? 2 : 1)) void delta_grad_kernel(GradArgs p) {
  using Lds = GradLds<T, DKB, KEPT>;
  constexpr int PK = KEPT, PI = PLANES<T>, DKP = Lds::DKP, PLANE = L * DKP * 2, TOK = Lds::TOK, STA = Lds::STA, W = DKB, THREADS = 64 * W;
  constexpr bool PAIR = !std::is_same_v<T, bf16_t>;
  extern __shared__ __align__(1024) char lds[];
  char *areaA = lds, *areaB = lds + Lds::A;
  float* kkm = (float*)(lds + Lds::IMAGE);
  float *dpm = (float*)areaB, *dam = (float*)(areaB + Lds::KK);
  float* red = (float*)(areaB + Lds::B);  // [4][W][L], [L]
  float* wred = red + (4 * W + 1) * L;    // [64]
  double* bs = (double*)(wred + 64);
  float* betas = (float*)(bs + L);        // [L], then row sums [2][L]
  float* rows = betas + L;
  float* ksc = rows + 2 * L;              // the scales of K's rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, gq = lane >> 4;
  const int64_t part = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int bh = (int)(part / p.chunks), chunk = (int)(part - (int64_t)bh * p.chunks);
  const int b = bh / p.NH, h = bh - b * p.NH, t0 = chunk * L;
  const int64_t image = ((int64_t)b * (p.NH / p.group) + h / p.group) * p.chunks + chunk;
  const Factors* f = p.prep.f + part;
  const int blocks = p.kept.blocks;
  const int64_t blk0 = part * blocks;

  // ---- Blocks of columns have scales of their own (exponents here); a product's sum over the columns takes the largest of its
  // two scales' product, and one operand of a smaller block the factor that is left.
  const float* const scales[5] = {p.kept.dhs + blk0, p.kept.zs + blk0, p.kept.us + blk0, p.kept.s0s + blk0, p.kept.dss + blk0};
  enum { DH_S, Z_S, U_DS, DH_U, Z_U, S_DS, SUMS };
  auto products = [&](const float (&of)[5], int (&to)[SUMS]) {
    int e[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) e[i] = (int)(__float_as_uint(of[i]) >> 23) - 127;
    to[DH_S] = e[0] + e[3];
    to[Z_S] = e[1] + e[3];
    to[U_DS] = e[2] + e[4];
    to[DH_U] = e[0] + e[2];
    to[Z_U] = e[1] + e[2];
    to[S_DS] = e[3] + e[4];
  };
  auto power = [](int e) { return e < -126 ? 0.f : __uint_as_float((uint32_t)(e + 127) << 23); };  // e <= 0
  int top[SUMS];
#pragma unroll
  for (int i = 0; i < SUMS; ++i) top[i] = -1000;
  for (int j = lane; j < blocks; j += 64) {
    int x[SUMS];
    const float of[5] = {scales[0][j], scales[1][j], scales[2][j], scales[3][j], scales[4][j]};
    products(of, x);
#pragma unroll
    for (int i = 0; i < SUMS; ++i) top[i] = max(top[i], x[i]);
  }
#pragma unroll
  for (int i = 0; i < SUMS; ++i) top[i] = uniform((int)wave_max_all((float)(top[i] + 1000)) - 1000);
  if (tid < L) {
    bs[tid] = f->b[tid];
    betas[tid] = f->beta[tid];
    ksc[tid] = power_of(f->k[tid]);
  }

  // ---- staging: pieces of 16 bytes, through registers
  constexpr int TOK_PIECES = 3 * PK * 256, TOK_PER = (TOK_PIECES + THREADS - 1) / THREADS, STA_PER = 2 * PK;  // of each state
  u32x4 tok[TOK_PER], sta[2][STA_PER];
  float coming[2][5];  // the scales of a step's two blocks
  // V of a token and 8 neighbours: wave w has tokens 16 w + r (and 16 (w + 2) + r where there are two)
  constexpr int MTS = 4 / (W < 4 ? W : 4);
  struct alignas(16) Eight { T e[8]; };
  Eight v8[MTS];
  // Bases that are the same for all and 32-bit offsets: addresses of each lane's own would leave no registers for what is under way.
  const char* const vrows = (const char*)((const T*)p.v + b * p.vs[0] + h * p.vs[1] + t0 * p.vs[2]);
  char* const dvrows = (char*)((T*)p.dv + ((int64_t)bh * p.S + t0) * p.DV);
  const int last = p.S - 1 - t0;
  auto load_v = [&](int step) {
    if (wave >= 4) return;
    const int n = 32 * step + 8 * gq;
#pragma unroll
    for (int x = 0; x < MTS; ++x) {
      const char* from = vrows + (uint32_t)(min(16 * (wave + x * W) + r, last) * (int)p.vs[2]) * (uint32_t)sizeof(T);
      if (p.wide_v) {  // past the last column the first ones, against Z's zeros
        v8[x] = *(const Eight*)(from + (uint32_t)(n < p.DV ? n : 0) * (uint32_t)sizeof(T));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v8[x].e[e] = n + e < p.DV ? ((const T*)from)[n + e] : from_f32<T>(0.f);
      }
    }
  };
  auto tok_of = [&](const f16_t* kept) { return (const char*)(kept + kept_at(part, blocks, 0, PK, L)); };
  auto sta_of = [&](const f16_t* kept) { return (const char*)(kept + kept_at(part, blocks, 0, PK, DKP)); };
  auto load = [&](int step) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < 5; ++i) coming[half][i] = scales[i][2 * step + half];
    const uint32_t tok_step = step * (uint32_t)(2 * PK * 16 * L * 2), sta_step = step * (uint32_t)(2 * PK * 16 * DKP * 2);
#pragma unroll
    for (int i = 0; i < TOK_PER; ++i) {
      const int at = min(i * THREADS + tid, TOK_PIECES - 1), mat = uniform(at / (PK * 256)), rest = at - mat * (PK * 256);
      const int pl = rest >> 8, row = (rest >> 3) & 31, piece = rest & 7;
      const uint32_t off = ((row >> 4) * PK + pl) * (16 * L * 2) + (row & 15) * (L * 2) + piece * 16;
      tok[i] = __builtin_bit_cast(u32x4, load16(tok_of(mat == 0 ? p.kept.dh : mat == 1 ? p.kept.z : p.kept.u), tok_step + off));
    }
#pragma unroll
    for (int mat = 0; mat < 2; ++mat)
#pragma unroll
      for (int i = 0; i < STA_PER; ++i) {
        const int at = (i / PK) * THREADS + tid, pl = i % PK, row = at / (DKP / 8), piece = at % (DKP / 8);
        const uint32_t off = ((row >> 4) * PK + pl) * (16 * DKP * 2) + (row & 15) * (DKP * 2) + piece * 16;
        sta[mat][i] = __builtin_bit_cast(u32x4, load16(sta_of(mat ? p.kept.ds : p.kept.s0), sta_step + off));
      }
  };
  float ss_dot = 0.f;  // <dS, S_0>
  auto store = [&] {
#pragma unroll
    for (int i = 0; i < TOK_PER; ++i) {
      const int at = i * THREADS + tid;
      if (at >= TOK_PIECES) continue;
      const int plane = at >> 8, row = (at >> 3) & 31, piece = at & 7;
      *(u32x4*)(areaA + plane * TOK + row * 128 + ((piece ^ (row & 7)) << 4)) = tok[i];
    }
#pragma unroll
    for (int mat = 0; mat < 2; ++mat)
#pragma unroll
      for (int i = 0; i < STA_PER; ++i) {
        const int at = (i / PK) * THREADS + tid, pl = i % PK, row = at / (DKP / 8), piece = at % (DKP / 8);
        *(u32x4*)(areaA + 3 * PK * TOK + (mat * PK + pl) * STA + row * (DKP * 2) + ((piece ^ (row & 7)) << 4)) = sta[mat][i];
      }
#pragma unroll
    for (int i = 0; i < STA_PER; i += PK) {
      const f16x8 a = __builtin_bit_cast(f16x8, sta[0][i]), d = __builtin_bit_cast(f16x8, sta[1][i]);
      f16x8 al = {}, dl = {};
      if constexpr (PK == 2) {
        al = __builtin_bit_cast(f16x8, sta[0][i + 1]);
        dl = __builtin_bit_cast(f16x8, sta[1][i + 1]);
      }
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x = fmaf((float)a[e] + (float)al[e], (float)d[e] + (float)dl[e], x);
      int e[SUMS];
      products(coming[i / PK], e);  // THREADS pieces are a block
      ss_dot = fmaf(x, power(e[S_DS] - top[S_DS]), ss_dot);
    }
  };
  // operands, k = the 32 columns: tokens 16 mt .. of matrix mat (0 dH, 1 Z, 2 U); DQK's columns 16 t .. of S_0 (0), dS (1)
  const int k0 = 8 * gq + (r >> 2);
  auto tok_frag = [&](int mat, int pl, int mt) {
    const char* base = areaA + (mat * PK + pl) * TOK + (mt & 1) * 8;
    const int piece = 4 * (mt >> 1) + (r & 3);
    return __builtin_bit_cast(f16x8, mfma::tr_pair(base + k0 * 128 + ((piece ^ (k0 & 7)) << 4),
                                                   base + (k0 + 4) * 128 + ((piece ^ ((k0 + 4) & 7)) << 4)));
  };
  auto sta_frag = [&](int mat, int pl, int t) {
    const char* base = areaA + 3 * PK * TOK + (mat * PK + pl) * STA + (t & 1) * 8;
    const int piece = 4 * (t >> 1) + (r & 3);
    return __builtin_bit_cast(f16x8, mfma::tr_pair(base + k0 * (DKP * 2) + ((piece ^ (k0 & 7)) << 4),
                                                   base + (k0 + 4) * (DKP * 2) + ((piece ^ ((k0 + 4) & 7)) << 4)));
  };

  f32x4 g1[2][4], g2[2][4], g3[2][4];  // dH S_0^T, Z S_0^T, U dS^T, turned
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) g1[t][mt] = g2[t][mt] = g3[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  // 10 tiles of dP and 10 of Z U^T: job, job + W, ..
  constexpr int JOBS = (20 + W - 1) / W;
  f32x4 jobs[JOBS];
  int job_mat[JOBS], job_i[JOBS], job_j[JOBS];
#pragma unroll
  for (int x = 0; x < JOBS; ++x) {
    jobs[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int job = min(x * W + wave, 19), tile = job % 10, i = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3;
    job_mat[x] = job / 10;
    job_i[x] = i;
    job_j[x] = tile - i * (i + 1) / 2;
  }
  float zv[MTS] = {};  // Z.V of tokens 16 mt + r

  const int steps = blocks / 2;
  load(0);
  load_v(0);
  for (int step = 0; step < steps; ++step) {
    lds_barrier();
    store();
    float of[5];  // a lane's 8 columns are of one block
#pragma unroll
    for (int i = 0; i < 5; ++i) of[i] = gq >> 1 ? coming[1][i] : coming[0][i];
    lds_barrier();
    // dV = beta Z, and Z.V: a lane has 8 neighbours of a token
    if (wave < 4) {
#pragma unroll
      for (int x = 0; x < MTS; ++x) {
        const int mt = wave + x * W, t = t0 + 16 * mt + r, n = 32 * step + 8 * gq;
        const f16x8 z = tok_frag(1, 0, mt);
        f16x8 zl = {};
        if constexpr (PK == 2) zl = tok_frag(1, 1, mt);
        if (t < p.S) {
          float zf[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) zf[e] = ((float)z[e] + (float)zl[e]) * of[1];
          const float beta = betas[16 * mt + r];
          char* const to = dvrows + (uint32_t)((t - t0) * p.DV + n) * (uint32_t)sizeof(T);
          f32x4 dv[2];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            zv[x] = fmaf(zf[e], to_f32(v8[x].e[e]), zv[x]);
            dv[e >> 2][e & 3] = beta * zf[e];
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const Four<T> o = rounded4<T>(dv[q]);
            if (p.wide_v) {
              if (n < p.DV) ((Four<T>*)to)[q] = o;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n + 4 * q + e < p.DV) ((T*)to)[4 * q + e] = o.e[e];
            }
          }
        }
      }
    }
    int factor[SUMS];
    products(of, factor);
    _Float16 by[SUMS];
#pragma unroll
    for (int i = 0; i < SUMS; ++i) by[i] = (_Float16)power(factor[i] - top[i]);
    __builtin_amdgcn_sched_barrier(0);
    load(step + 1 < steps ? step + 1 : step);  // past the last step that one again
    load_v(step + 1 < steps ? step + 1 : step);
    f16x8 s0[PK][2], ds[PK][2];
#pragma unroll
    for (int pl = 0; pl < PK; ++pl)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s0[pl][t] = sta_frag(0, pl, 2 * wave + t);
        ds[pl][t] = sta_frag(1, pl, 2 * wave + t);
      }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      const f16x8 d = tok_frag(0, 0, mt) * by[DH_S], z = tok_frag(1, 0, mt) * by[Z_S], u = tok_frag(2, 0, mt) * by[U_DS];
      f16x8 dl, zl, ul;
      if constexpr (PK == 2) {
        dl = tok_frag(0, 1, mt) * by[DH_S];
        zl = tok_frag(1, 1, mt) * by[Z_S];
        ul = tok_frag(2, 1, mt) * by[U_DS];
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (PK == 2) {
          g1[t][mt] = mfma(s0[1][t], d, g1[t][mt]);
          g1[t][mt] = mfma(s0[0][t], dl, g1[t][mt]);
          g2[t][mt] = mfma(s0[1][t], z, g2[t][mt]);
          g2[t][mt] = mfma(s0[0][t], zl, g2[t][mt]);
          g3[t][mt] = mfma(ds[1][t], u, g3[t][mt]);
          g3[t][mt] = mfma(ds[0][t], ul, g3[t][mt]);
        }
        g1[t][mt] = mfma(s0[0][t], d, g1[t][mt]);
        g2[t][mt] = mfma(s0[0][t], z, g2[t][mt]);
        g3[t][mt] = mfma(ds[0][t], u, g3[t][mt]);
      }
    }
#pragma unroll
    for (int x = 0; x < JOBS; ++x) {
      const _Float16 share = job_mat[x] ? by[Z_U] : by[DH_U];
      const f16x8 a = tok_frag(job_mat[x], 0, job_i[x]), u = tok_frag(2, 0, job_j[x]) * share;
      if constexpr (PK == 2) {
        jobs[x] = mfma(tok_frag(job_mat[x], 1, job_i[x]), u, jobs[x]);
        jobs[x] = mfma(a, tok_frag(2, 1, job_j[x]) * share, jobs[x]);
      }
      jobs[x] = mfma(a, u, jobs[x]);
    }
  }
  // K and the wave's rows of P are on their way meanwhile
  u32x4 image_regs[4 * PI];
  auto bring = [&](const char* img) {
#pragma unroll
    for (int i = 0; i < 4 * PI; ++i) image_regs[i] = *(const u32x4*)(img + image * (PI * PLANE) + (i * THREADS + tid) * 16);
  };
  auto put_image = [&] {
#pragma unroll
    for (int i = 0; i < 4 * PI; ++i) *(u32x4*)(areaA + (i * THREADS + tid) * 16) = image_regs[i];
  };
  static_assert(4 * THREADS * 16 == PLANE);
  bring(p.prep.k);
  constexpr int ROWS = L / W;
  f16_t ph[ROWS], pl[ROWS];
  const f16_t* pf = p.prep.p + part * (2 * FRAG_PLANE);
#pragma unroll
  for (int x = 0; x < ROWS; ++x) {
    // P's operand order: lane (i % 16) + 16 of 4 columns, halves of 16 of each 32
    const int i = x * W + wave, j = lane;
    const int at = (2 * (i >> 4) + (j >> 5)) * 512 + ((i & 15) + 16 * ((j >> 2) & 3)) * 8 + ((j >> 4) & 1) * 4 + (j & 3);
    ph[x] = pf[at];
    pl[x] = pf[at + FRAG_PLANE];
  }
  lds_barrier();

  // ---- dP, dA to LDS; K beside
#pragma unroll
  for (int x = 0; x < JOBS; ++x) {
    if (x * W + wave >= 20) continue;
    float* to = job_mat[x] ? dam : dpm;
    const int sc = job_mat[x] ? top[Z_U] : top[DH_U];
#pragma unroll
    for (int e = 0; e < 4; ++e) to[(16 * job_i[x] + 4 * gq + e) * GLD + 16 * job_j[x] + r] = ldexpf(job_mat[x] ? -jobs[x][e] : jobs[x][e], sc);
  }
  put_image();
  bring(p.prep.q);
  lds_barrier();
#pragma unroll
  for (int x = 0; x < (10 + W - 1) / W; ++x) {
    const int tile = x * W + wave;
    if (tile >= 10) continue;
    const int i = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, j = tile - i * (i + 1) / 2;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DKB; ++s) {
      const f16x8 a = rows_frag<DKP>(areaA, i, s, r, gq), c = rows_frag<DKP>(areaA, j, s, r, gq);
      if constexpr (PI == 2) {
        y = mfma(rows_frag<DKP>(areaA + PLANE, i, s, r, gq), c, y);
        y = mfma(a, rows_frag<DKP>(areaA + PLANE, j, s, r, gq), y);
      }
      y = mfma(a, c, y);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) kkm[(16 * i + 4 * gq + e) * GLD + 16 * j + r] = y[e] * (ksc[16 * i + 4 * gq + e] * ksc[16 * j + r]);
  }
  // sum over DQK's columns of this wave of K or Q times a turned accumulator, into red[slot][wave][token]
  auto dots = [&](const f32x4 (&g)[2][4], int slot) {
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      float x = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int tile = 2 * wave + t;
        const char* at = areaA + piece_at<DKP>(16 * mt + r, 4 * (tile >> 1) + gq) + (tile & 1) * 8;
        const f16x4 a = *(const f16x4*)at;
        f16x4 al = {};
        if constexpr (PI == 2) al = *(const f16x4*)(at + PLANE);
#pragma unroll
        for (int e = 0; e < 4; ++e) x = fmaf((float)a[e] + (float)al[e], g[t][mt][e], x);
      }
      x += __shfl_xor(x, 16, 64);
      x += __shfl_xor(x, 32, 64);
      if (gq == 0) red[(slot * W + wave) * L + 16 * mt + r] = x;
    }
  };
  dots(g2, 0);  // k_i.(Z S_0^T)_i
  dots(g3, 1);  // k_j.(U dS^T)_j
  lds_barrier();

  // ---- each pair of tokens: wave w has rows w, w + W, .., a lane a column
  // dQ takes scale D o dP against K's planes, dK its transpose against Q's and E + E^T against K's: the scales of the planes' rows enter
  // here, and dK's two have one scale between them, so that their sum is in one unit.  (A chunk without a pair of tokens has zeros for E, one without
  // dH for dP: in units of its own the other part could be past float32's range.)
  float dps[ROWS], ee[ROWS], col = 0.f, mx[2] = {0.f, 0.f};
  const double bj = bs[lane];
  // a lane's token's; a row's are read from its lane
  const float kj = ksc[lane], qj = power_of(f->qs[lane]), pj = power_of(f->p[lane]);
  auto of_row = [&](float x, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)); };
#pragma unroll
  for (int x = 0; x < ROWS; ++x) {
    const int i = x * W + wave, j = lane;
    const bool on = j <= i, below = j < i;
    const float dec = on ? exp_of(bs[i] - bj) : 0.f;
    const float pv = on ? ((float)ph[x] + (float)pl[x]) * of_row(pj, i) : 0.f;
    const float dp = on ? dpm[i * GLD + j] : 0.f, da = below ? dam[i * GLD + j] : 0.f, beta = betas[i];
    const float nij = below ? dec * kkm[i * GLD + j] : 0.f;
    const float bb = wave_sum_dpp(da * nij), pp = wave_sum_dpp(dp * pv);
    if (lane == 63) {
      rows[i] = pp;
      rows[L + i] = bb;
    }
    col += fmaf(dp, pv, beta * (da * nij));
    dps[x] = p.scale * dec * dp;
    ee[x] = da * beta * dec;
    mx[0] = fmaxf(mx[0], fabsf(dps[x]) * kj);
    mx[1] = fmaxf(mx[1], fmaxf(fabsf(dps[x]) * of_row(qj, i), fabsf(ee[x]) * fmaxf(kj, of_row(kj, i))));
  }
  red[(2 * W + wave) * L + lane] = col;
  const float m0 = wave_max_all(mx[0]), m1 = wave_max_all(mx[1]), dot = wave_sum(ss_dot);
  if (lane == 0) {
    wred[wave] = m0;
    wred[8 + wave] = m1;
    wred[16 + wave] = dot;
  }
#pragma unroll
  for (int x = 0; x < MTS; ++x) {
    if (wave >= 4) continue;
    float y = zv[x];
    y += __shfl_xor(y, 16, 64);
    y += __shfl_xor(y, 32, 64);
    if (gq == 0) red[4 * W * L + 16 * (wave + x * W) + r] = y;
  }
  lds_barrier();  // dP and dA have been read: their place takes the operands
  mx[0] = mx[1] = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    mx[0] = fmaxf(mx[0], wred[w]);
    mx[1] = fmaxf(mx[1], wred[8 + w]);
  }
  const Pow2 sq = pow2_for(mx[0]), sk = pow2_for(mx[1]);
  // rows of 64 in f16, each 32 turned, piece p of row i at p ^ (i % 8): scale D o dP, its transpose, E + E^T
  constexpr int MAT = L * L * 2;
  auto put = [&](int mat, int i, int j, float x) {
    char* at = areaB + mat * MAT + i * 128 + (((4 * (j >> 5) + ((j >> 2) & 3)) ^ (i & 7)) << 4) + ((j >> 4) & 1) * 8 + (j & 3) * 2;
    const _Float16 hi = (_Float16)x;
    *(_Float16*)at = hi;
    if constexpr (PAIR) *(_Float16*)(at + 3 * MAT) = (_Float16)(x - (float)hi);
  };
#pragma unroll
  for (int x = 0; x < ROWS; ++x) {
    const int i = x * W + wave, j = lane;
    put(0, i, j, dps[x] * kj * sq.up);
    put(1, j, i, dps[x] * of_row(qj, i) * sk.up);
    if (j <= i) put(2, i, j, ee[x] * kj * sk.up);
    if (j < i) put(2, j, i, ee[x] * of_row(kj, i) * sk.up);
  }
  lds_barrier();
  auto pair_frag = [&](int mat, int pl, int mt, int s) {
    const int i = 16 * mt + r;
    return *(const f16x8*)(areaB + (pl * 3 + mat) * MAT + i * 128 + (((4 * s + gq) ^ (i & 7)) << 4));
  };
  // acc[t][mt] += (columns of the image in LDS)^T mat
  auto add = [&](f32x4 (&acc)[2][4], int mat) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f16x8 a = columns_frag<DKP>(areaA, 2 * wave + t, s, r, gq);
        f16x8 al;
        if constexpr (PI == 2) al = columns_frag<DKP>(areaA + PLANE, 2 * wave + t, s, r, gq);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const f16x8 x = pair_frag(mat, 0, mt, s);
          if constexpr (PI == 2) acc[t][mt] = mfma(al, x, acc[t][mt]);
          if constexpr (PAIR) acc[t][mt] = mfma(a, pair_frag(mat, 1, mt, s), acc[t][mt]);
          acc[t][mt] = mfma(a, x, acc[t][mt]);
        }
      }
  };
  // dK's parts with the states (in g3 from here)
  f32x4 accq[2][4], acck[2][4];
#pragma unroll
  for (int mt = 0; mt < 4; ++mt) {
    const double bt = bs[16 * mt + r];
    const float fo = ldexpf(exp_of(bs[L - 1] - bt), top[U_DS]), fb = ldexpf(betas[16 * mt + r] * exp_of(bt), top[Z_S]);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      g3[t][mt] = g3[t][mt] * fo - g2[t][mt] * fb;
      accq[t][mt] = acck[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  add(accq, 0);
  add(acck, 2);
  lds_barrier();
  put_image();
  lds_barrier();
  add(acck, 1);
  dots(g1, 3);  // q_i.(dH S_0^T)_i
  // ---- out
  {
    float fq[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) fq[mt] = ldexpf(p.scale * exp_of(bs[16 * mt + r]), top[DH_S]);
    auto write = [&](auto type, auto whole) {
      using O = decltype(type);
      const int d = 32 * wave + 4 * gq;
      const int64_t at = ((int64_t)bh * p.S + t0 + r) * p.DK + d;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if (t0 + 16 * mt + r >= p.S) continue;
        O *const q = (O*)p.dq + at + (int64_t)(16 * mt) * p.DK, *const k = (O*)p.dk + at + (int64_t)(16 * mt) * p.DK;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Four<O> oq = rounded4<O>(g1[t][mt] * fq[mt] + accq[t][mt] * sq.down), ok = rounded4<O>(g3[t][mt] + acck[t][mt] * sk.down);
          if constexpr (decltype(whole)::value) {
            if (d + 16 * t < p.DK) {
              *(Four<O>*)(q + 16 * t) = oq;
              *(Four<O>*)(k + 16 * t) = ok;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + 16 * t + e < p.DK) {
                q[16 * t + e] = oq.e[e];
                k[16 * t + e] = ok.e[e];
              }
          }
        }
      }
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (p.group == 1) p.DK % 4 == 0 ? write(T{}, Yes{}) : write(T{}, No{});
    else p.DK % 4 == 0 ? write(float{}, Yes{}) : write(float{}, No{});
  }
  lds_barrier();
  // ---- the gates, a lane a token
  if (wave != 0) return;
  float kz = 0.f, ks = 0.f, qd = 0.f, cl = 0.f, dss = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    kz += red[(0 * W + w) * L + lane];
    ks += red[(1 * W + w) * L + lane];
    cl += red[(2 * W + w) * L + lane];
    qd += red[(3 * W + w) * L + lane];
    dss += wred[16 + w];
  }
  const float ckz = ldexpf(f->in[lane] * kz, top[Z_S]);    // in and out have K's scale, which kz and ks lack
  const float sj = ldexpf(f->out[lane] * ks, top[U_DS]);
  const float qi = ldexpf(f->q[lane] * qd, top[DH_S]);
  const float beta = betas[lane];
  const float dbeta = red[4 * W * L + lane] - ckz + rows[L + lane];
  float db = rows[lane] + beta * rows[L + lane] - cl - sj + qi - beta * ckz;
  const float sums = wave_sum(sj) + ldexpf(f->all * dss, top[S_DS]);
  if (lane == 63) db += sums;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float above = __shfl_down(db, o, 64);
    if (lane + o < 64) db += above;
  }
  const int token = t0 + lane;
  if (token >= p.S) return;
  const int64_t at = (int64_t)bh * p.S + token;
  auto gates = [&](auto type) {
    using G = decltype(type);
    ((G*)p.dg)[at] = from_f32<G>(db);
    ((G*)p.dbeta)[at] = from_f32<G>(dbeta);
  };
  switch (p.gate_dtype) {
    case XL_DTYPE_F32: gates(0.f); break;
    case XL_DTYPE_BF16: gates(bf16_t{}); break;
    default: gates(f16_t{}); break;
  }
}

// ------------------------------------------------------------------------------------------------ shared heads
// to [B NHK, S DK] = sums over the group of from [B NHK, group, S DK]
template <typename T>
__global__ __launch_bounds__(256) void delta_join_kernel(const float* __restrict__ from, T* __restrict__ to, int group, int64_t per,
                                                         int64_t count) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const int64_t head = i / per;
    const float* at = from + head * group * per + (i - head * per);
    float x = 0.f;
    for (int j = 0; j < group; ++j) x += at[j * per];
    to[i] = from_f32<T>(x);
  }
}

// ------------------------------------------------------------------------------------------------ host
int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

struct Layout {
  int64_t prep, tok, sta, scales, partial;  // bytes of one of each
  int blocks;
  explicit Layout(const Shape& s) {
    blocks = 2 * ((s.DV + 31) / 32);
    prep = up256((int64_t)prep_bytes(s, true));
    tok = up256(s.parts() * blocks * s.kept() * 16 * L * 2);
    sta = up256(s.parts() * blocks * s.kept() * 16 * s.dkp() * 2);
    scales = up256(s.parts() * blocks * 4);
    partial = s.NH == s.NHK ? 0 : up256((int64_t)s.B * s.NH * s.S * s.DK * 4);
  }
  int64_t bytes() const { return prep + 3 * tok + 2 * sta + 5 * scales + 2 * partial; }
};

hipError_t launch(const void* kern, int64_t grid, int grid_y, int threads, int64_t lds, void* arg, hipStream_t st) {
  void* args[] = {arg};
  hipError_t e = lds > 65536 ? hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) : hipSuccess;
  return e != hipSuccess ? e : hipLaunchKernel(kern, dim3((unsigned)grid, grid_y), dim3(threads), args, (unsigned)lds, st);
}

template <typename T, int KEPT>
int backward(const Shape& s, const void* v, const void* dh, const float* dc_last, void* dq, void* dk, void* dv, void* dg,
             void* dbeta, float* dc0, const float* c0, const Prep& prep, const Kept& kept, float* dqp, float* dkp, hipStream_t st,
             const char* who) {
  const int group = s.NH / s.NHK, chunks = s.chunks();
  TurnArgs turn{dh, kept, s.S, s.DV, chunks, s.DV % 8 == 0 && ((uintptr_t)dh & 15) == 0};
  hipError_t e = launch((const void*)delta_turn_kernel<T, KEPT>, s.parts(), (kept.blocks + 3) / 4, 256, 0, &turn, st);
  if (e == hipSuccess)
    if (const int rc = launch_scan(s, v, c0, nullptr, nullptr, prep, &kept, st, who)) return rc;
  constexpr int S8 = PLANES<T> == 2 ? 1 : 2;
  const int stages = s.dkp() == 256 ? S8 : 2;
  // A lone wave a block where two workgroups a CU (one, if no two fit) take all blocks, else four blocks a workgroup.  us of whole calls,
  // 2048 tokens, lone waves and fours: bf16 128 x 256, 256 blocks 252, 277; 512 433, 454; 768 626, 572; 1024 755, 689; 64 x 256, 512
  // blocks 346, 357; 1024 637, 577; 256 x 512, 512 blocks 597, 548; float32 128 x 256, 512 blocks of 1024 tokens 362, 349; f16
  // 128 x 256, 256 blocks 420, 468; 512 748, 785; 768 1040, 983; 256 x 512, 512 blocks 1188, 1151.
  const int64_t scan_lds = stages * 2 * s.image_bytes() + 2 * 2048;
  const int waves = (int64_t)s.B * s.NH * kept.blocks <= (scan_lds <= 80 * 1024 ? 512 : 256) ? 1 : 4;
  const int slices = (kept.blocks + waves - 1) / waves;
  BackArgs back{dc_last, dc0, prep, kept, s.NH, group, s.DK, s.DV, chunks, slices};
  const void* kern =
      waves == 4 ? s.dkp() == 64    ? (const void*)delta_back_kernel<T, 2, 2, 4, KEPT>
                   : s.dkp() == 128 ? (const void*)delta_back_kernel<T, 4, 2, 4, KEPT> : (const void*)delta_back_kernel<T, 8, S8, 4, KEPT>
      : s.dkp() == 64    ? (const void*)delta_back_kernel<T, 2, 2, 1, KEPT>
        : s.dkp() == 128 ? (const void*)delta_back_kernel<T, 4, 2, 1, KEPT> : (const void*)delta_back_kernel<T, 8, S8, 1, KEPT>;
  if (e == hipSuccess)
    e = launch(kern, (int64_t)s.B * s.NH * slices, 1, waves == 1 ? 128 : 64 * waves, scan_lds, &back, st);
  GradArgs grad{v, {s.vs[0], s.vs[1], s.vs[2]}, group == 1 ? dq : (void*)dqp, group == 1 ? dk : (void*)dkp, dv, dg, dbeta, prep, kept,
                s.NH, group, s.S, s.DK, s.DV, chunks, s.dtype_gates, s.scale, false};
  constexpr int VW = 16 / sizeof(T);
  grad.wide_v = s.DV % 8 == 0 && ((s.vs[0] | s.vs[1] | s.vs[2]) % VW) == 0 && (((uintptr_t)v | (uintptr_t)dv) & 15) == 0;
  const int lds = s.dkp() == 64 ? GradLds<T, 2, KEPT>::BYTES : s.dkp() == 128 ? GradLds<T, 4, KEPT>::BYTES : GradLds<T, 8, KEPT>::BYTES;
  kern = s.dkp() == 64 ? (const void*)delta_grad_kernel<T, 2, KEPT> : s.dkp() == 128 ? (const void*)delta_grad_kernel<T, 4, KEPT>
                                                                                    : (const void*)delta_grad_kernel<T, 8, KEPT>;
  if (e == hipSuccess) e = launch(kern, s.parts(), 1, s.dkp() * 2, lds, &grad, st);
  if (e == hipSuccess && group > 1) {
    const int64_t per = (int64_t)s.S * s.DK, count = (int64_t)s.B * s.NHK * per;
    const unsigned grid = (unsigned)((count + 255) / 256 < 8192 ? (count + 255) / 256 : 8192);
    delta_join_kernel<T><<<grid, 256, 0, st>>>(dqp, (T*)dq, group, per, count);
    delta_join_kernel<T><<<grid, 256, 0, st>>>(dkp, (T*)dk, group, per, count);
  }
  if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
  return check_launch(who);
}

}  // namespace
}  // namespace delta
}  // namespace xl

extern "C" size_t xl_gated_delta_chunkwise_bwd_workspace_size_gates(int B, int NH, int NHK, int S, int DQK, int DV, int dtype_qkv,
                                                                    int dtype_gates) {
  using namespace xl;
  delta::Shape s{B, NH, NHK, S, DQK, DV, {}, {}, {}, 1.f, dtype_qkv, dtype_gates};
  if (delta::check_shape("xl_gated_delta_chunkwise_bwd_workspace_size", s) != XL_OK) return 0;
  return S == 0 ? 0 : (size_t)delta::Layout(s).bytes();
}

// float32 gates keep pairs whatever q, k and v are
extern "C" size_t xl_gated_delta_chunkwise_bwd_workspace_size(int B, int NH, int NHK, int S, int DQK, int DV, int dtype_qkv) {
  return xl_gated_delta_chunkwise_bwd_workspace_size_gates(B, NH, NHK, S, DQK, DV, dtype_qkv, XL_DTYPE_F32);
}

extern "C" int xl_gated_delta_chunkwise_bwd(const void* q, const void* k, const void* v, const int64_t* strides, const void* g,
                                            const void* beta, const float* c0, const void* dh, const float* dc_last, void* dq,
                                            void* dk, void* dv, void* dg, void* dbeta, float* dc0, int B, int NH, int NHK,
                                            int S, int DQK, int DV, float scale, int dtype_qkv, int dtype_gates,
                                            void* workspace, size_t workspace_bytes, void* stream) {
  using namespace xl;
  const char* who = "xl_gated_delta_chunkwise_bwd";
  clear_error();
  delta::Shape s{B, NH, NHK, S, DQK, DV, {}, {}, {}, scale, dtype_qkv, dtype_gates};
  if (const int rc = delta::check_shape(who, s)) return rc;
  if (S == 0) return set_error(XL_ERR_INVALID_ARG, "%s: no tokens", who);
  if (!q || !k || !v || !g || !beta || !dh || !dq || !dk || !dv || !dg || !dbeta)
    return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15)
    return set_error(XL_ERR_INVALID_ARG, "%s: dq, dk and dv must be 16-byte aligned", who);
  if (dc0 && dc0 == dc_last) return set_error(XL_ERR_INVALID_ARG, "%s: dc0 must not alias dc_last", who);
  const delta::Layout lay(s);
  if (!workspace || workspace_bytes < (size_t)lay.bytes() || ((uintptr_t)workspace & 255))
    return set_error(XL_ERR_WORKSPACE, "%s: the workspace must be %zu bytes, 256-byte aligned", who, (size_t)lay.bytes());
  if (const int rc = delta::set_strides(s, strides, who)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  const delta::Prep prep = delta::prep_at(s, true, ws);
  char* at = ws + lay.prep;
  auto take = [&](int64_t bytes) {
    char* x = at;
    at += bytes;
    return x;
  };
  delta::Kept kept{};
  kept.u = (f16_t*)take(lay.tok);
  kept.z = (f16_t*)take(lay.tok);
  kept.dh = (f16_t*)take(lay.tok);
  kept.s0 = (f16_t*)take(lay.sta);
  kept.ds = (f16_t*)take(lay.sta);
  for (float** x : {&kept.us, &kept.zs, &kept.dhs, &kept.s0s, &kept.dss}) *x = (float*)take(lay.scales);
  kept.blocks = lay.blocks;
  float *dqp = (float*)take(lay.partial), *dkp = (float*)take(lay.partial);
  if (const int rc = delta::launch_prep(s, q, k, g, beta, prep, true, st, who)) return rc;
  auto run = [&](auto t, auto planes) {
    return delta::backward<decltype(t), decltype(planes)::value>(s, v, dh, dc_last, dq, dk, dv, dg, dbeta, dc0, c0, prep, kept, dqp, dkp, st, who);
  };
  using Pairs = std::integral_constant<int, 2>;
  if (dtype_qkv == XL_DTYPE_F32) return run(float{}, Pairs{});
  if (dtype_qkv == XL_DTYPE_F16) return run(f16_t{}, Pairs{});
  return s.kept() == 2 ? run(bf16_t{}, Pairs{}) : run(bf16_t{}, std::integral_constant<int, 1>{});
}
