// Gated delta rule by chunks, second kernel: the scan over a head's chunks (delta.h has the formulas).
//
// Every 16 columns of V, U and the state go through the sequence by themselves: heads times DV / 16 chains, each chunk's step of
// which is bound by the time of dependent products, reductions and LDS exchanges, not by bytes or operations.  Where such
// blocks are many, a wave takes one, four of them share the chunk's images in LDS (delta_scan_wave_kernel).  Where they are
// few, up to four waves take one (delta_scan_kernel): a wave has its part of the state's rows (float32 registers) and as
// large a part of a chunk's tokens.  Per chunk:
//
//   1  K S and Q S over the wave's rows, all tokens; the others' tokens go to LDS
//   2  R = diag(beta) (V - diag(c) K S) of the wave's tokens, to LDS as f16 planes
//   3  U = T R of the wave's tokens, to LDS as f16 planes, decayed for the state and as it is for H
//   4  S = c_L S + K^T U of the wave's rows; H = Q S + P U of the wave's tokens
//
// The images of K and Q come to LDS straight from memory, K a chunk ahead, Q into the place of this chunk's when it has been read;
// in delta_scan_kernel by a wave of its own (a load into LDS that has to queue stops its wave).  T, P and V of the next chunk wait in
// registers.  H is formed turned (columns down, tokens across): a lane holds four neighbours of a row.  Measured (bf16): 2 x 4096 tokens
// of 8 heads of 128 x 256 138 to 145 us, 2.2 a chunk; 4 x 8192 of 8 heads of 256 x 512 580 to 627, 4.5 to 4.9 a chunk.
#include "delta.h"

namespace xl {
namespace delta {
namespace {

struct ScanArgs {
  const void* v;
  int64_t vs[3];
  const float* c0;
  void* h;
  float* c_last;
  Prep prep;
  Kept kept;
  int NH, group, S, DK, DV, chunks, slices;
};

// LDS of a scan's workgroup: KST stages of K, one of Q, two chunks' factors, and the exchanges
template <int DKB, int PK, int PARTS, int KST, bool WITH_Q, bool WIDE_U>
struct ScanLds {
  static constexpr int IMG = PK * L * DKB * 32 * 2;
  static constexpr int Q = KST * IMG, FACTORS = Q + (WITH_Q ? IMG : 0);
  // sums of the others' parts (then of Q S), R, U decayed, U, scales
  static constexpr int SUMS = FACTORS + 2 * 1024, R = SUMS + 4 * PARTS * 1024, UD = R + 4096, U = UD + 4096, SCALES = U + (WIDE_U ? 4096 : 2048);
  static constexpr int BYTES = SCALES + 64;
};

// KEPT: U and the state before each chunk are kept for the backward, in as many planes, and nothing else is written; 0: the forward.
// PAIR: the outputs' products too are of pairs (f16, whose own rounding is a single plane's, and float32).  bf16's h, off by up to
// 2^-8 by its own rounding, takes P, U and the state in one plane there, 2^-11 each (pairs: 4 to 12 % of a call); its U and state are
// formed of pairs.
template <typename T, int DKB, int PARTS, int KST, int KEPT>
__global__ __launch_bounds__(64 * PARTS + 64) void delta_scan_kernel(ScanArgs p) {
  constexpr bool STATES = KEPT != 0;
  constexpr int DKP = DKB * 32, PK = PLANES<T>, PLANE = L * DKP * 2, IMG = PK * PLANE;
  constexpr int TPW = 4 / PARTS, NB = DKB / PARTS;  // a wave's tiles of 16 tokens, its 32s of DQK
  constexpr bool PAIR = !STATES && !std::is_same_v<T, bf16_t>;
  using Lds = ScanLds<DKB, PK, PARTS, KST, !STATES, PAIR>;
  static_assert(DKB % PARTS == 0 && Lds::BYTES <= 160 * 1024);
  extern __shared__ __align__(1024) char lds[];
  const int lane = threadIdx.x & 63, part = uniform(threadIdx.x >> 6);
  const int r = lane & 15, gq = lane >> 4;
  const int all = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int bh = uniform(all / p.slices), block = all - bh * p.slices, b = uniform(bh / p.NH), h = bh - b * p.NH;
  const int64_t image0 = ((int64_t)b * uniform(p.NH / p.group) + uniform(h / p.group)) * p.chunks, part0 = (int64_t)bh * p.chunks;
  const int n0 = block * 16, n = n0 + r;
  const T* v = (const T*)p.v + b * p.vs[0] + h * p.vs[1];
  T* ho = (T*)p.h + (int64_t)bh * p.S * p.DV;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_char*)lds;
  float* const scales = (float*)(lds + Lds::SCALES);  // [R, U, state, U decayed][part]
  // sums over part `from`'s rows of token tile mt (its owner's own too: to leave those out took branches that cost more)
  auto sums_at = [&](int mt, int from) { return (f32x4*)(lds + Lds::SUMS) + (mt * PARTS + from) * 64 + lane; };
  auto sum_of = [&](int mt) {
    f32x4 x[PARTS];
#pragma unroll
    for (int i = 0; i < PARTS; ++i) x[i] = *sums_at(mt, i);
#pragma unroll
    for (int i = 1; i < PARTS; ++i) x[0] += x[i];
    return x[0];
  };

  if (part == PARTS) {  // brings the images: a wave whose load into LDS has to queue stands still
    auto fetch = [&](const char* images, int chunk, int to) {
      const char* img = images + (image0 + chunk) * (int64_t)IMG;
#pragma unroll
      for (int i = 0; i < IMG / 1024; ++i) to_lds(lds_at + to + i * 1024, i * 1024 + lane * 16, img);
    };
    auto fetch_factors = [&](int chunk) { to_lds(lds_at + Lds::FACTORS + (chunk & 1) * 1024, lane * 16, p.prep.f + part0 + chunk); };
    fetch(p.prep.k, 0, 0);
    if constexpr (!STATES) fetch(p.prep.q, 0, Lds::Q);
    fetch_factors(0);
    lds_barrier();  // the other waves' barriers: of the first state,
    for (int c = 0; c < p.chunks; ++c) {
      wait_loads();
      lds_barrier();  // a chunk's begin,
      if (KST == 2 && c + 1 < p.chunks) fetch(p.prep.k, c + 1, ((c + 1) & 1) * IMG);
      lds_barrier();  // the partial sums: Q has been read,
      if (c + 1 < p.chunks) {
        if constexpr (!STATES) fetch(p.prep.q, c + 1, Lds::Q);
        fetch_factors(c + 1);
      }
      lds_barrier();  // R,
      lds_barrier();  // U
      if (KST == 1) {
        lds_barrier();
        if (c + 1 < p.chunks) fetch(p.prep.k, c + 1, 0);
      }
    }
    return;
  }
  // Tokens 16 mt + 4 gq + e of column n, mt of this wave.  Past the last token the last one is read again (beta is 0 there),
  // past the last column the last one: those columns are computed and not written.
  const int nc = n < p.DV ? n : p.DV - 1, row_step = (int)p.vs[2];
  T vn[TPW][4];
  uint32_t v_at[TPW][4];
#pragma unroll
  for (int x = 0; x < TPW; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v_at[x][e] = (uint32_t)((16 * (part * TPW + x) + 4 * gq + e) * row_step + nc) * (uint32_t)sizeof(T);
  auto load_v = [&](int chunk) {
    const int t0 = chunk * L;
    if (t0 + L > p.S) {  // the last chunk, once
#pragma unroll
      for (int x = 0; x < TPW; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = 16 * (part * TPW + x) + 4 * gq + e, last = p.S - 1 - t0;
          v_at[x][e] = (uint32_t)((t < last ? t : last) * row_step + nc) * (uint32_t)sizeof(T);
        }
    }
    const char* base = (const char*)(v + t0 * p.vs[2]);
#pragma unroll
    for (int x = 0; x < TPW; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) vn[x][e] = *(const T*)(base + v_at[x][e]);
  };
  // T's and P's rows of the wave's tokens, both halves of k
  f16x8 th[TPW][2], tl[TPW][2], ph[TPW][2], pl[TPW][2], ph_next[TPW][2], pl_next[TPW][2];
  auto load_rows = [&](const f16_t* from, f16x8 (&to)[TPW][2]) {
#pragma unroll
    for (int x = 0; x < TPW; ++x)
#pragma unroll
      for (int s = 0; s < 2; ++s) to[x][s] = load16(from + (2 * (part * TPW + x) + s) * 512, lane * 16);
  };
  float all_next, t_next;  // the next chunk's factors that are not in LDS
  uint8_t p_next[TPW];
  auto load_t = [&](int chunk) {
    const f16_t* from = p.prep.t + (part0 + chunk) * (2 * FRAG_PLANE);
    load_rows(from, th);
    load_rows(from + FRAG_PLANE, tl);
    const Factors* f = p.prep.f + part0 + chunk;
    all_next = f->all;
    t_next = f->t;
    if constexpr (!STATES) {
#pragma unroll
      for (int x = 0; x < TPW; ++x) p_next[x] = f->p[16 * (part * TPW + x) + r];
    }
  };
  auto load_p = [&](int chunk) {
    const f16_t* from = p.prep.p + (part0 + chunk) * (2 * FRAG_PLANE);
    load_rows(from, ph_next);
    if constexpr (PAIR) load_rows(from + FRAG_PLANE, pl_next);
  };

  f32x4 st[2 * NB];  // the wave's rows of the state, times 1 / st_down (the same for all parts)
#pragma unroll
  for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * (2 * NB * part + t) + 4 * gq + e;
      st[t][e] = p.c0 && d < p.DK ? p.c0[((int64_t)bh * p.DK + d) * p.DV + nc] : 0.f;
    }
  auto largest = [&](const float* of) {
    float m = of[0];
#pragma unroll
    for (int i = 1; i < PARTS; ++i) m = fmaxf(m, of[i]);
    return __int_as_float(uniform(__float_as_int(m)));
  };
  float st_down, most = state_max(st);
  if (lane == 0) scales[2 * PARTS + part] = most;
  __syncthreads();
  {
    const Pow2 sc = pow2_for(largest(scales + 2 * PARTS), STATE);
    st_down = sc.down;
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) st[t] *= sc.up;
  }

  load_v(0);
  load_t(0);
  if constexpr (!STATES) load_p(0);
  const bool kept = STATES && block < p.kept.blocks;
  const uint32_t h_at = (uint32_t)(r * p.DV + 4 * gq) * sizeof(T);
  Four<T> o[TPW];  // the chunk's H, written when the next one's loads have been waited for
  auto store_h = [&](int chunk) {
    const int t0 = chunk * L;
    T* const to = ho + (int64_t)t0 * p.DV + n0;
    const bool whole = t0 + L <= p.S && n0 + 16 <= p.DV && p.DV % 4 == 0;
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      const int mt = part * TPW + x;
      if (whole) {
        *(Four<T>*)((char*)(to + (int64_t)(16 * mt) * p.DV) + h_at) = o[x];
      } else if (t0 + 16 * mt + r < p.S) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n0 + 4 * gq + e < p.DV) to[(int64_t)(16 * mt + r) * p.DV + 4 * gq + e] = o[x].e[e];
      }
    }
  };
  for (int c = 0; c < p.chunks; ++c) {
    // The chunk's only wait for memory: T, V and P left a good part of a chunk ago.
    wait_loads();
    lds_barrier();
    const int stage = KST == 2 ? (c & 1) * IMG : 0, next = c + 1 < p.chunks ? c + 1 : c;
    if constexpr (!STATES) {
      if (c) store_h(c - 1);
#pragma unroll
      for (int x = 0; x < TPW; ++x)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          ph[x][s] = ph_next[x][s];
          if constexpr (PAIR) pl[x][s] = pl_next[x][s];
        }
    }
    const char *ki = lds + stage, *qi = lds + Lds::Q;
    const Factors* f = (const Factors*)(lds + Lds::FACTORS + (c & 1) * 1024);

    // ---- 1: K S, and Q S turned, over the wave's rows
    f32x4 ks[4], hs[STATES ? 1 : 4], in[TPW], bv[TPW], out[TPW];
    float fq[TPW], fp[TPW];
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      const int mt = part * TPW + x;
      in[x] = *(const f32x4*)&f->back[16 * mt + 4 * gq];
      bv[x] = *(const f32x4*)&f->beta[16 * mt + 4 * gq];
      out[x] = *(const f32x4*)&f->out[16 * mt + 4 * gq];
      if constexpr (!STATES) {
        fq[x] = f->q[16 * mt + r];
        fp[x] = power_of(p_next[x]);
      }
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      ks[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (!STATES) hs[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      const int sb = part * NB + s;
      f16x8 k[PK][4], q[STATES ? 1 : PK][4], hi, lo;
#pragma unroll
      for (int pl = 0; pl < PK; ++pl)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) k[pl][mt] = rows_frag<DKP>(ki + pl * PLANE, mt, sb, r, gq);
      if constexpr (!STATES) {
#pragma unroll
        for (int pl = 0; pl < PK; ++pl)
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) q[pl][mt] = rows_frag<DKP>(qi + pl * PLANE, mt, sb, r, gq);
      }
      __builtin_amdgcn_sched_barrier(0);  // every read under way at once, here and below
      split8(st[2 * s], st[2 * s + 1], hi, lo);
      if constexpr (STATES) {
        if (kept) {
          f16_t* to = p.kept.s0 + kept_at(part0 + c, p.kept.blocks, block, KEPT, DKP);
          *(f16x8*)((char*)to + r * (DKP * 2) + gq * 16 + sb * 64) = hi;
          if constexpr (KEPT == 2) *(f16x8*)((char*)(to + 16 * DKP) + r * (DKP * 2) + gq * 16 + sb * 64) = lo;
        }
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if constexpr (PK == 2) ks[mt] = mfma(k[1][mt], hi, ks[mt]);
        ks[mt] = mfma(k[0][mt], hi, ks[mt]);
        ks[mt] = mfma(k[0][mt], lo, ks[mt]);
      }
      if constexpr (!STATES) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          if constexpr (PK == 2) hs[mt] = mfma(hi, q[1][mt], hs[mt]);
          hs[mt] = mfma(hi, q[0][mt], hs[mt]);
          if constexpr (PAIR) hs[mt] = mfma(lo, q[0][mt], hs[mt]);
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) *sums_at(mt, part) = ks[mt];
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      in[x] *= st_down;
#pragma unroll
      for (int e = 0; e < 4; ++e) bv[x][e] *= to_f32(vn[x][e]);
      if constexpr (!STATES) fq[x] *= st_down;
    }
    const float keep = all_next, t_scale = t_next;
    most = state_max(st) * st_down;
    if (lane == 0) scales[2 * PARTS + part] = most;
    lds_barrier();
    // ---- 2: R
    f32x4 rr[TPW];
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      const f32x4 sum = sum_of(part * TPW + x);
#pragma unroll
      for (int e = 0; e < 4; ++e) rr[x][e] = fmaf(-in[x][e], sum[e], bv[x][e]);
    }
    load_v(next);
    if constexpr (!STATES) load_p(next);
    const Pow2 rs = pow2_for(wave_max_all(abs_max(rr)));
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      f16x4 hi, lo;
      split4(rr[x], rs.up, hi, lo);
      *((f16x8*)(lds + Lds::R) + (part * TPW + x) * 64 + lane) = join(hi, lo);
    }
    if (lane == 0) scales[part] = rs.down;
    lds_barrier();
    // ---- 3: U
    f16x8 raw[4], rh[2], rl[2];
    float of[PARTS];
    auto read_scales = [&](int from, float (&to)[PARTS]) {
#pragma unroll
      for (int i = 0; i < PARTS; ++i) to[i] = scales[from * PARTS + i];
    };
    auto read4 = [&](int at) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = *((const f16x8*)(lds + at) + i * 64 + lane);
    };
    read_scales(0, of);
    read4(Lds::R);
    __builtin_amdgcn_sched_barrier(0);
    // of a part's scale to the largest's
    auto shifts = [&](const float (&of)[PARTS], float down, _Float16 (&by)[PARTS]) {
#pragma unroll
      for (int i = 0; i < PARTS; ++i) by[i] = ratio(__int_as_float(uniform(__float_as_int(of[i]))), down);
    };
    auto planes = [&](const _Float16 (&by)[PARTS], f16x8 (&hi)[2], f16x8 (&lo)[2]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f16x8 a = raw[2 * s] * by[2 * s / TPW], b = raw[2 * s + 1] * by[(2 * s + 1) / TPW];
        hi[s] = join(f16x4{a[0], a[1], a[2], a[3]}, f16x4{b[0], b[1], b[2], b[3]});
        lo[s] = join(f16x4{a[4], a[5], a[6], a[7]}, f16x4{b[4], b[5], b[6], b[7]});
      }
    };
    _Float16 by[PARTS];
    const float r_down = largest(of);
    shifts(of, r_down, by);
    planes(by, rh, rl);
    f32x4 u[TPW], w[TPW];
    const float back = t_scale * r_down;
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      f32x4 y = {0.f, 0.f, 0.f, 0.f}, y2 = y;
      y = mfma(tl[x][0], rh[0], y);
      y2 = mfma(th[x][0], rl[0], y2);
      if (part * TPW + x >= 2) {
        y = mfma(tl[x][1], rh[1], y);
        y2 = mfma(th[x][1], rl[1], y2);
        y = mfma(th[x][1], rh[1], y);
      }
      y2 = mfma(th[x][0], rh[0], y2);
      u[x] = (y + y2) * back;
      w[x] = u[x] * out[x];
    }
    load_t(next);
    const Pow2 us = pow2_for(wave_max_all(abs_max(u))), ws = pow2_for(wave_max_all(abs_max(w)));
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      const int mt = part * TPW + x;
      f16x4 hi, lo;
      split4(w[x], ws.up, hi, lo);
      *((f16x8*)(lds + Lds::UD) + mt * 64 + lane) = join(hi, lo);
      if constexpr (!STATES) {
        split4(u[x], us.up, hi, lo);
        if constexpr (PAIR) *((f16x8*)(lds + Lds::U) + mt * 64 + lane) = join(hi, lo);
        else *((f16x4*)(lds + Lds::U) + mt * 64 + lane) = hi;
      }
    }
    if (lane == 0) {
      scales[PARTS + part] = us.down;
      scales[3 * PARTS + part] = ws.down;
    }
    if constexpr (!STATES) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) *sums_at(mt, part) = hs[mt];
    }
    lds_barrier();
    // ---- 4: the state
    f16x8 kc[2 * NB][PK][2], raw_u[PAIR ? 4 : 1];
    f16x4 half_u[PAIR || STATES ? 1 : 4];
    f32x4 qs[STATES ? 1 : TPW];
    float of_u[PARTS], of_s[PARTS], of_w[PARTS];
    read_scales(1, of_u);
    read_scales(2, of_s);
    read_scales(3, of_w);
    read4(Lds::UD);
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
      for (int pl = 0; pl < PK; ++pl)
#pragma unroll
        for (int s = 0; s < 2; ++s) kc[t][pl][s] = columns_frag<DKP>(ki + pl * PLANE, 2 * NB * part + t, s, r, gq);
    if constexpr (!STATES) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (PAIR) raw_u[i] = *((const f16x8*)(lds + Lds::U) + i * 64 + lane);
        else half_u[i] = *((const f16x4*)(lds + Lds::U) + i * 64 + lane);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    const float u_down = largest(of_u);
    // U decayed is below 2^15 of its scale
    const Pow2 sc = pow2_for(fmaxf(largest(of_s) * keep, largest(of_w) * 32767.f), STATE);
    // U decayed from its parts' scales to the state's, in two steps of 2^-24 at most: as one f16 factor what is 2^-25 or less (writes of 2^-17 of the
    // state and below) would be 0
    f16x8 wh[2], wl[2];
    _Float16 by2[PARTS];
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const float x = of_w[i] * sc.up;
      by[i] = (_Float16)fmaxf(x, 0x1p-24f);
      by2[i] = (_Float16)fminf(x * 0x1p24f, 1.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = raw[i] * by[i / TPW];
    planes(by2, wh, wl);
    shifts(of_u, u_down, by);
    if constexpr (!STATES) {
#pragma unroll
      for (int x = 0; x < TPW; ++x) qs[x] = sum_of(part * TPW + x);
    }
    const float up = keep * st_down * sc.up;
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) {
      f32x4 y = {0.f, 0.f, 0.f, 0.f}, y2 = y;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if constexpr (PK == 2) y2 = mfma(kc[t][1][s], wh[s], y2);
        y2 = mfma(kc[t][0][s], wl[s], y2);
        y = mfma(kc[t][0][s], wh[s], y);
      }
      st[t] = fma4(st[t], up, y + y2);
    }
    if constexpr (STATES) {
      if (kept) {
        const _Float16 by = ratio(us.down, u_down);
#pragma unroll
        for (int x = 0; x < TPW; ++x) {
          const int mt = part * TPW + x;
          f16x4 hi, lo;
          split4(u[x], us.up, hi, lo);
          char* to = (char*)(p.kept.u + kept_at(part0 + c, p.kept.blocks, block, KEPT, L)) + r * (L * 2) + (mt >> 1) * 64 + gq * 16 + (mt & 1) * 8;
          *(f16x4*)to = hi * by;
          if constexpr (KEPT == 2) *(f16x4*)(to + 16 * L * 2) = lo * by;
        }
        if (lane == 0 && part == 0) {
          const int64_t at = (part0 + c) * p.kept.blocks + block;
          p.kept.us[at] = u_down;
          p.kept.s0s[at] = st_down;
        }
      }
    } else {  // ---- H
      f16x8 uh[2], ul[2];
      if constexpr (PAIR) {
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = raw_u[i];
        planes(by, uh, ul);
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) uh[s] = join(half_u[2 * s] * by[2 * s / TPW], half_u[2 * s + 1] * by[(2 * s + 1) / TPW]);
      }
#pragma unroll
      for (int x = 0; x < TPW; ++x) {
        const int mt = part * TPW + x;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        y = mfma(uh[0], ph[x][0], y);
        if constexpr (PAIR) {
          y = mfma(ul[0], ph[x][0], y);
          y = mfma(uh[0], pl[x][0], y);
        }
        if (mt >= 2) {
          y = mfma(uh[1], ph[x][1], y);
          if constexpr (PAIR) {
            y = mfma(ul[1], ph[x][1], y);
            y = mfma(uh[1], pl[x][1], y);
          }
        }
        o[x] = rounded4<T>(y * (fp[x] * u_down) + qs[x] * fq[x]);
      }
    }
    st_down = sc.down;
    if (KST == 1) lds_barrier();
  }
  if constexpr (!STATES) store_h(p.chunks - 1);
  wait_loads();
  if (p.c_last && n < p.DV) {
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 16 * (2 * NB * part + t) + 4 * gq + e;
        if (d < p.DK) p.c_last[((int64_t)bh * p.DK + d) * p.DV + n] = st[t][e] * st_down;
      }
  }
}

// A block by one wave, W blocks a workgroup.
template <typename T, int DKB, int STAGES, int KEPT>
__global__ __launch_bounds__(256, 1) void delta_scan_wave_kernel(ScanArgs p) {
  constexpr bool STATES = KEPT != 0;
  constexpr int W = 4, DKP = DKB * 32, PK = PLANES<T>, PLANE = L * DKP * 2, IMG = PK * PLANE, STAGE = (STATES ? 1 : 2) * IMG;
  constexpr int FACTORS = 1280;  // of a chunk's Factors, in LDS
  constexpr bool PAIR = STATES ? KEPT == 2 : !std::is_same_v<T, bf16_t>;
  extern __shared__ __align__(1024) char lds[];  // STAGES of K and Q; two chunks' factors
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int r = lane & 15, gq = lane >> 4;
  const int all = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int bh = uniform(all / p.slices), slice = all - bh * p.slices, b = uniform(bh / p.NH), h = bh - b * p.NH;
  const int64_t image0 = ((int64_t)b * uniform(p.NH / p.group) + uniform(h / p.group)) * p.chunks, part0 = (int64_t)bh * p.chunks;
  const int n0 = (slice * W + wave) * 16, n = n0 + r;
  const T* v = (const T*)p.v + b * p.vs[0] + h * p.vs[1];
  T* ho = (T*)p.h + (int64_t)bh * p.S * p.DV;

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
      to_lds(lds_at + stage * STAGE + (i + wave) * 1024, (i + wave) * 1024 + lane * 16, STATES || i < IMG / 1024 ? ki : qi);
    }
  };
  auto fetch_factors = [&](int chunk) {
    if (wave >= 2) return;  // 1.25 KB: the second wave's KB lies over the first's
    const uint32_t from = wave * (FACTORS - 1024);
    to_lds(lds_at + STAGES * STAGE + (chunk & 1) * FACTORS + from, from + lane * 16, p.prep.f + part0 + chunk);
  };
  // Rows 16 mt + 4 gq + e of column n.  Past the last token the last one is read again (beta is 0 there), past the last column the
  // last one: those columns are computed and not written.
  const int nc = n < p.DV ? n : p.DV - 1, row_step = (int)p.vs[2];
  T vn[4][4];
  uint32_t v_at[4][4];
#pragma unroll
  for (int mt = 0; mt < 4; ++mt)
#pragma unroll
    for (int e = 0; e < 4; ++e) v_at[mt][e] = (uint32_t)((16 * mt + 4 * gq + e) * row_step + nc) * (uint32_t)sizeof(T);
  auto load_v = [&](int chunk) {
    const int t0 = chunk * L;
    if (t0 + L > p.S) {  // the last chunk, once
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = 16 * mt + 4 * gq + e, last = p.S - 1 - t0;
          v_at[mt][e] = (uint32_t)((t < last ? t : last) * row_step + nc) * (uint32_t)sizeof(T);
        }
    }
    const char* base = (const char*)(v + t0 * p.vs[2]);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) vn[mt][e] = *(const T*)(base + v_at[mt][e]);
  };

  f32x4 st[2 * DKB];  // the state times 1 / st_down
#pragma unroll
  for (int t = 0; t < 2 * DKB; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * t + 4 * gq + e;
      st[t][e] = p.c0 && d < p.DK ? p.c0[((int64_t)bh * p.DK + d) * p.DV + nc] : 0.f;
    }
  float st_down;
  {
    const Pow2 sc = pow2_for(state_max(st), STATE);
    st_down = sc.down;
#pragma unroll
    for (int t = 0; t < 2 * DKB; ++t) st[t] *= sc.up;
  }

  // T, P and V of the next chunk wait in registers, K, Q and the factors in LDS.  What is loaded past the last chunk is that one's
  // again.
  f16x8 th[LOWER], tl[LOWER], ph[LOWER], pl[PAIR ? LOWER : 1];
  auto load_t = [&](int chunk) {
    const f16_t* from = p.prep.t + (part0 + chunk) * (2 * FRAG_PLANE);
    load_lower(from, lane, th);
    load_lower(from + FRAG_PLANE, lane, tl);
  };
  auto load_p = [&](int chunk) {
    const f16_t* from = p.prep.p + (part0 + chunk) * (2 * FRAG_PLANE);
    load_lower(from, lane, ph);
    if constexpr (PAIR) load_lower(from + FRAG_PLANE, lane, pl);
  };
#pragma unroll
  for (int s = 0; s < DKB; ++s) fetch(0, 0, s);
  fetch_factors(0);
  load_v(0);
  load_t(0);
  if constexpr (!STATES) load_p(0);
  const int block = n0 / 16;
  const bool kept = STATES && block < p.kept.blocks;
  const uint32_t h_at = (uint32_t)(r * p.DV + 4 * gq) * sizeof(T);
  for (int c = 0; c < p.chunks; ++c) {
    // The chunk's only wait for memory: the compiler does not count the loads into LDS, and its waits for a register behind them were
    // for some of them too (666 us, 627 so).
    wait_loads();
    lds_barrier();
    const int stage = STAGES == 2 ? c & 1 : 0, next = c + 1 < p.chunks ? c + 1 : c;
    if (next != c) fetch_factors(next);
    const char *ki = lds + stage * STAGE, *qi = ki + IMG;
    const Factors* f = (const Factors*)(lds + STAGES * STAGE + (c & 1) * FACTORS);

    // ---- K S, and Q S turned: the operands of the next 32 of DQK are read under the products of these
    struct Rows {
      f16x8 k[PK][4], q[STATES ? 1 : PK][4];
    };
    auto read = [&](Rows& to, int s) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int pl = 0; pl < PK; ++pl) {
          to.k[pl][mt] = rows_frag<DKP>(ki + pl * PLANE, mt, s, r, gq);
          if constexpr (!STATES) to.q[pl][mt] = rows_frag<DKP>(qi + pl * PLANE, mt, s, r, gq);
        }
    };
    f32x4 ks[4], hs[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) ks[mt] = hs[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    Rows rows[2];
    read(rows[0], 0);
    f32x4 in[4], bv[4], out[4];
    float fq[4], fp[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      in[mt] = *(const f32x4*)&f->back[16 * mt + 4 * gq] * st_down;
      bv[mt] = *(const f32x4*)&f->beta[16 * mt + 4 * gq];
#pragma unroll
      for (int e = 0; e < 4; ++e) bv[mt][e] *= to_f32(vn[mt][e]);
      out[mt] = *(const f32x4*)&f->out[16 * mt + 4 * gq];
      if constexpr (!STATES) {
        fq[mt] = f->q[16 * mt + r] * st_down;
        fp[mt] = power_of(f->p[16 * mt + r]);
      }
    }
    const float keep = f->all, t_scale = f->t;
    f16x8 sh[2], sl[2];
    split8(st[0], st[1], sh[0], sl[0]);
#pragma unroll
    for (int s = 0; s < DKB; ++s) {
      if (s + 1 < DKB) read(rows[(s + 1) & 1], s + 1);
      if (STAGES == 2) fetch(next, stage ^ 1, s);
      __builtin_amdgcn_sched_barrier(0);
      const Rows& x = rows[s & 1];
      const f16x8 hi = sh[s & 1], lo = sl[s & 1];
      if (s + 1 < DKB) split8(st[2 * s + 2], st[2 * s + 3], sh[(s + 1) & 1], sl[(s + 1) & 1]);
      if constexpr (STATES) {
        if (kept) {
          f16_t* to = p.kept.s0 + kept_at(part0 + c, p.kept.blocks, block, KEPT, DKP) + r * DKP + s * 32 + gq * 8;
          *(f16x8*)to = hi;
          if constexpr (KEPT == 2) *(f16x8*)(to + 16 * DKP) = lo;
        }
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if constexpr (PK == 2) ks[mt] = mfma(x.k[1][mt], hi, ks[mt]);
        ks[mt] = mfma(x.k[0][mt], hi, ks[mt]);
        if constexpr (!STATES) {
          if constexpr (PK == 2) hs[mt] = mfma(hi, x.q[1][mt], hs[mt]);
          hs[mt] = mfma(hi, x.q[0][mt], hs[mt]);
        }
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        ks[mt] = mfma(x.k[0][mt], lo, ks[mt]);
        if constexpr (PAIR && !STATES) hs[mt] = mfma(lo, x.q[0][mt], hs[mt]);
      }
      interleave<8 + (STATES ? 0 : 4) + (PK == 2 ? 4 : 0)>();
      __builtin_amdgcn_sched_barrier(0);
    }
    // ---- R
    f32x4 rr[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) rr[mt][e] = fmaf(-in[mt][e], ks[mt][e], bv[mt][e]);
    load_v(next);
    const Pow2 rs = pow2_for(wave_max_all(abs_max(rr)));
    f16x8 rh[2], rl[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) split8<true>(rr[2 * s], rr[2 * s + 1], rs.up, rh[s], rl[s]);
    // ---- U
    f32x4 u[4];
    const float back = t_scale * rs.down;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) u[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < LOWER; ++i) u[lower_mt(i)] = mfma(th[i], rh[lower_s(i)], u[lower_mt(i)]);
#pragma unroll
    for (int i = 0; i < LOWER; ++i) u[lower_mt(i)] = mfma(tl[i], rh[lower_s(i)], u[lower_mt(i)]);
#pragma unroll
    for (int i = 0; i < LOWER; ++i) u[lower_mt(i)] = mfma(th[i], rl[lower_s(i)], u[lower_mt(i)]);
    load_t(next);
    const float most = abs_max(st) * (st_down * keep);  // a lane's, not needed before w
    // the first operands of the state's product
    constexpr int AHEAD = 4;
    f16x8 columns[AHEAD][PK][2];
    auto read_columns = [&](int t) {
#pragma unroll
      for (int pl = 0; pl < PK; ++pl)
#pragma unroll
        for (int s = 0; s < 2; ++s) columns[t % AHEAD][pl][s] = columns_frag<DKP>(ki + pl * PLANE, t, s, r, gq);
    };
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) read_columns(t);
    f32x4 w[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      u[mt] *= back;
      w[mt] = u[mt] * out[mt];
    }
    const Pow2 us = pow2_for(wave_max_all(abs_max(u)));
    const Pow2 ws = pow2_for(wave_max_all(fmaxf(abs_max(w), most)), STATE);
    f16x8 uh[2], ul[2], wh[2], wl[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      split8<PAIR>(u[2 * s], u[2 * s + 1], us.up, uh[s], ul[s]);
      split8<true>(w[2 * s], w[2 * s + 1], ws.up, wh[s], wl[s]);
    }
    f32x4 x[4];
    if constexpr (STATES) {
      if (kept) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          f16_t* to = p.kept.u + kept_at(part0 + c, p.kept.blocks, block, KEPT, L) + r * L + s * 32 + gq * 8;
          *(f16x8*)to = uh[s];
          if constexpr (KEPT == 2) *(f16x8*)(to + 16 * L) = ul[s];
        }
        if (lane == 0) {
          const int64_t at = (part0 + c) * p.kept.blocks + block;
          p.kept.us[at] = us.down;
          p.kept.s0s[at] = st_down;
        }
      }
    } else {  // ---- P U
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) x[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < LOWER; ++i) {
        f32x4& y = x[lower_mt(i)];
        y = mfma(uh[lower_s(i)], ph[i], y);
        if constexpr (PAIR) {
          y = mfma(ul[lower_s(i)], ph[i], y);
          y = mfma(uh[lower_s(i)], pl[i], y);
        }
      }
      load_p(next);
    }
    // ---- the state
    const float up = keep * st_down * ws.up;
    st_down = ws.down;
#pragma unroll
    for (int t = 0; t < 2 * DKB; ++t) {
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if constexpr (PK == 2) y = mfma(columns[t % AHEAD][1][s], wh[s], y);
        y = mfma(columns[t % AHEAD][0][s], wl[s], y);
        y = mfma(columns[t % AHEAD][0][s], wh[s], y);
      }
      st[t] = fma4(st[t], up, y);
      if (t + AHEAD < 2 * DKB) read_columns(t + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
    // ---- H
    if constexpr (!STATES) {
      const int t0 = c * L;
      T* const to = ho + (int64_t)t0 * p.DV + n0;
      const bool whole = t0 + L <= p.S && n0 + 16 <= p.DV && p.DV % 4 == 0;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const Four<T> o = rounded4<T>(x[mt] * (fp[mt] * us.down) + hs[mt] * fq[mt]);
        if (whole) {
          *(Four<T>*)((char*)(to + (int64_t)(16 * mt) * p.DV) + h_at) = o;
        } else if (t0 + 16 * mt + r < p.S) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + 4 * gq + e < p.DV) to[(int64_t)(16 * mt + r) * p.DV + 4 * gq + e] = o.e[e];
        }
      }
    }
    if (STAGES == 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (next != c) {
#pragma unroll
        for (int s = 0; s < DKB; ++s) fetch(next, 0, s);
      }
    }
  }
  wait_loads();
  if (p.c_last && n < p.DV) {
#pragma unroll
    for (int t = 0; t < 2 * DKB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 16 * t + 4 * gq + e;
        if (d < p.DK) p.c_last[((int64_t)bh * p.DK + d) * p.DV + n] = st[t][e] * st_down;
      }
  }
}

struct Choice {
  const void* kern;
  int threads, blocks, lds;  // threads of a workgroup, its blocks of 16 columns
};
// At most a block of columns a CU: by as many waves as there are 32s of DQK, up to 4.  More: one a wave, 4 a workgroup.  us of whole
// calls of bf16, 2048 tokens, both ways (waves of a block, a wave): 128 x 256, 256 blocks 91, 112; 512 171, 128; 1024 316, 165; 2048
// 613, 335; 64 x 256, 512 blocks 104, 98; 256 x 512, 512 blocks 181, 147; 1024 365, 180.
template <typename T, int DKB, int KEPT>
Choice choice(bool many) {
  constexpr bool STATES = KEPT != 0;
  constexpr int PK = PLANES<T>, KST = DKB == 8 && PK == 2 && !STATES ? 1 : 2;  // K's pairs twice and Q's do not fit
  constexpr int PARTS = DKB < 4 ? DKB : 4;
  constexpr bool PAIR = !STATES && !std::is_same_v<T, bf16_t>;
  if (many)
    return {(const void*)delta_scan_wave_kernel<T, DKB, KST, KEPT>, 256, 4, KST * (STATES ? 1 : 2) * PK * L * DKB * 64 + 2 * 1280};
  return {(const void*)delta_scan_kernel<T, DKB, PARTS, KST, KEPT>, 64 * PARTS + 64, 1,
          ScanLds<DKB, PK, PARTS, KST, !STATES, PAIR>::BYTES};
}
template <typename T, int KEPT>
Choice pick(int dkp, bool many) {
  return dkp == 64 ? choice<T, 2, KEPT>(many) : dkp == 128 ? choice<T, 4, KEPT>(many) : choice<T, 8, KEPT>(many);
}

}  // namespace

int launch_scan(const Shape& s, const void* v, const float* c0, void* h, float* c_last, const Prep& prep, const Kept* kept,
                hipStream_t st, const char* who) {
  ScanArgs a{v, {s.vs[0], s.vs[1], s.vs[2]}, c0, h, c_last, prep, {}, s.NH, s.NH / s.NHK, s.S, s.DK, s.DV, s.chunks(), 0};
  if (kept) a.kept = *kept;
  const int blocks = kept ? kept->blocks : (s.DV + 15) / 16;
  const bool many = (int64_t)s.B * s.NH * blocks > 256;
  Choice use{};
  auto choose = [&](auto t) {
    using T = decltype(t);
    if (!kept) use = pick<T, 0>(s.dkp(), many);
    else if (s.kept() == 2) use = pick<T, 2>(s.dkp(), many);
    else if constexpr (std::is_same_v<T, bf16_t>) use = pick<T, 1>(s.dkp(), many);
  };
  if (s.dtype == XL_DTYPE_F32) choose(float{});
  else if (s.dtype == XL_DTYPE_BF16) choose(bf16_t{});
  else choose(f16_t{});
  a.slices = (blocks + use.blocks - 1) / use.blocks;
  void* args[] = {&a};
  hipError_t e = hipFuncSetAttribute(use.kern, hipFuncAttributeMaxDynamicSharedMemorySize, use.lds);
  if (e == hipSuccess)
    e = hipLaunchKernel(use.kern, dim3((unsigned)((int64_t)s.B * s.NH * a.slices)), dim3(use.threads), args, (unsigned)use.lds, st);
  if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
  return check_launch(who);
}

}  // namespace delta
}  // namespace xl

extern "C" size_t xl_gated_delta_chunkwise_workspace_size(int B, int NH, int NHK, int S, int DQK, int DV, int dtype_qkv) {
  using namespace xl;
  delta::Shape s{B, NH, NHK, S, DQK, DV, {}, {}, {}, 1.f, dtype_qkv, dtype_qkv};
  if (delta::check_shape("xl_gated_delta_chunkwise_workspace_size", s) != XL_OK) return 0;
  return S == 0 ? 0 : delta::prep_bytes(s, false);
}

extern "C" int xl_gated_delta_chunkwise_fwd(const void* q, const void* k, const void* v, const int64_t* strides, const void* g,
                                            const void* beta, const float* c0, void* h, float* c_last, int B, int NH, int NHK,
                                            int S, int DQK, int DV, float scale, int dtype_qkv, int dtype_gates,
                                            void* workspace, size_t workspace_bytes, void* stream) {
  using namespace xl;
  const char* who = "xl_gated_delta_chunkwise_fwd";
  clear_error();
  delta::Shape s{B, NH, NHK, S, DQK, DV, {}, {}, {}, scale, dtype_qkv, dtype_gates};
  if (const int rc = delta::check_shape(who, s)) return rc;
  if (S == 0 && !c_last) return XL_OK;
  if (S == 0) return delta::launch_recurrent(s, q, k, v, g, beta, c0, h, c_last, (hipStream_t)stream, who);
  if (!q || !k || !v || !g || !beta || !h) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if ((uintptr_t)h & 15) return set_error(XL_ERR_INVALID_ARG, "%s: h must be 16-byte aligned", who);
  if (c0 && c0 == c_last) return set_error(XL_ERR_INVALID_ARG, "%s: c_last must not alias c0", who);
  const size_t need = delta::prep_bytes(s, false);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))
    return set_error(XL_ERR_WORKSPACE, "%s: the workspace must be %zu bytes, 256-byte aligned", who, need);
  if (const int rc = delta::set_strides(s, strides, who)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const delta::Prep prep = delta::prep_at(s, false, (char*)workspace);
  if (const int rc = delta::launch_prep(s, q, k, g, beta, prep, false, st, who)) return rc;
  return delta::launch_scan(s, v, c0, h, c_last, prep, nullptr, st, who);
}
