// Gated delta rule by chunks, first kernel: what of a chunk does not depend on the state (delta.h has the formulas).
//
// A workgroup of 4 waves takes one chunk of one head of q and k: it brings K and Q to f16 planes, each token at a power-of-two scale of
// its own (their images go to memory as the scans' LDS wants them), forms K K^T and Q K^T once, and for each head of v that shares them
// the sums of g (in float64: differences of sums of strong decays keep their bits), A, T = (I + A)^-1 and P.
//
// T by 16 x 16 blocks, in float32: each wave inverts one diagonal block by substitution (a lane a column), then walks down
// its block column, T_ij = -T_ii sum_l A_il T_lj, with v_mfma_f32_16x16x4_f32, whose result is the next one's operand as it
// stands.  Everything a scan reads as an operand (T, P) is written in operand order, 16 bytes a lane.
// A token of beta 0 has U = 0, whatever its values: its columns of A, T and P, which only U meets, are left out, so that padding does not set
// their scales (in the backward T's alone: dbeta needs the transposed ones).
//
// Large: bound by memory (bf16, 4 x 8192 tokens of 8 heads of 256: 144 to 152 us for 0.64 GB in and out, which a copy takes
// 124 for); few chunks: by the chain of one (13 chunks of 8 heads of 128: 12.8 us).
#include "delta.h"

namespace xl {
namespace delta {
namespace {

struct PrepArgs {
  const void *q, *k, *g, *beta;
  int64_t qs[3], ks[3];
  int NH, NHK, S, DK, chunks;
  float scale;
  int gate_dtype;
  bool wide;  // 16-byte loads of q and k
  Prep out;
};

constexpr int MLD = 68;  // row length of 64 x 64 float32 matrices in LDS

// 8 values as they lie; zeros past n
template <typename T>
struct Raw8 {
  u32x4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int from, int n, bool wide) {
  Raw8<T> x;
  if (wide && from + 8 <= n) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.w[i] = *(const u32x4*)(p + from + 4 * i);
  } else {
    struct V { T e[8]; } v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v.e[e] = from + e < n ? p[from + e] : from_f32<T>(0.f);
    x = __builtin_bit_cast(Raw8<T>, v);
  }
  return x;
}
template <typename T>
__device__ __forceinline__ void values8(const Raw8<T>& raw, float (&x)[8]) {
  struct V { T e[8]; };
  const V v = __builtin_bit_cast(V, raw);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f32(v.e[e]);
}

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// max over the workgroup of N values a thread
template <int N>
__device__ __forceinline__ void block_max(float (&m)[N], float (*red)[8]) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m[i] = wave_max_all(m[i]);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][i] = m[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) m[i] = fmaxf(fmaxf(red[0][i], red[1][i]), fmaxf(red[2][i], red[3][i]));
}

template <typename T, int DKB, bool BWD>
__global__ __launch_bounds__(256) void delta_prep_kernel(PrepArgs p) {
  constexpr int DKP = DKB * 32, PK = PLANES<T>, IMG = L * DKP * 2;
  extern __shared__ __align__(1024) char lds[];  // the images of K and Q; then A, T and P
  __shared__ double bs[L];
  __shared__ float betas[L], red[4][8];
  __shared__ float ksc[L], qsc[L];  // rows of K, Q = planes * these; 0 for rows of zeros
  float *Am = (float*)lds, *Tm = Am + L * MLD, *Pm = Tm + L * MLD;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, gq = lane >> 4;
  const int64_t img = blockIdx.x;
  const int bk = (int)(img / p.chunks), chunk = (int)(img - (int64_t)bk * p.chunks);
  const int b = bk / p.NHK, hk = bk - b * p.NHK, group = p.NH / p.NHK;
  const int t0 = chunk * L;

  // ---- K and Q: a row's 32 columns are one piece of 8 of each of 4 threads
  const int row = tid >> 2, c = tid & 3;
  Raw8<T> raw[2][DKB];  // both under way at once
  const bool there = t0 + row < p.S;  // past the last token: its row again, for zeros
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int64_t* st = which ? p.qs : p.ks;
    const T* from = (const T*)(which ? p.q : p.k) + b * st[0] + hk * st[1] + (int64_t)(there ? t0 + row : p.S - 1) * st[2];
#pragma unroll
    for (int s = 0; s < DKB; ++s) raw[which][s] = load8(from, 32 * s + 8 * c, p.DK, p.wide);
  }
  float gt = 0.f, bt = 0.f;
  auto load_gates = [&](int64_t bh) {
    const int64_t at = bh * p.S + (t0 + lane < p.S ? t0 + lane : p.S - 1);
    auto gates = [&](auto type) {
      using G = decltype(type);
      gt = to_f32(((const G*)p.g)[at]);
      bt = to_f32(((const G*)p.beta)[at]);
    };
    switch (p.gate_dtype) {
      case XL_DTYPE_F32: gates(0.f); break;
      case XL_DTYPE_BF16: gates(bf16_t{}); break;
      default: gates(f16_t{}); break;
    }
    if (t0 + lane >= p.S) gt = bt = 0.f;
  };
  load_gates((int64_t)b * p.NH + hk * group);
  float m2[2] = {0.f, 0.f};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int s = 0; s < DKB; ++s) {
      float x[8];
      values8(raw[which][s], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) m2[which] = fmaxf(m2[which], there ? fabsf(x[e]) : 0.f);
    }
    m2[which] = fmaxf(m2[which], __shfl_xor(m2[which], 1, 64));
    m2[which] = fmaxf(m2[which], __shfl_xor(m2[which], 2, 64));
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const Pow2 sc = m2[which] == 0.f ? Pow2{1.f, 0.f} : pow2_for(m2[which], 0);
    if (c == 0) (which ? qsc : ksc)[row] = sc.down;
    const float up = there ? sc.up : 0.f;
    char* to = lds + which * PK * IMG;
#pragma unroll
    for (int s = 0; s < DKB; ++s) {
      f16x8 hi, lo;
      float x[8];
      values8(raw[which][s], x);
      if (!there) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
      }
      split8<PK == 2>(x, up, hi, lo);
      // values 8 c + 0..3 and 4..7 of the 32: groups 2 c, 2 c + 1 of 4, the second four groups in the upper halves
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = piece_at<DKP>(row, 4 * s + ((2 * c + h) & 3)) + (c >> 1) * 8;
        const u32x4 uh = __builtin_bit_cast(u32x4, hi), ul = __builtin_bit_cast(u32x4, lo);
        *(u32x2*)(to + at) = u32x2{uh[2 * h], uh[2 * h + 1]};
        if constexpr (PK == 2) *(u32x2*)(to + IMG + at) = u32x2{ul[2 * h], ul[2 * h + 1]};
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    char* to = (which ? p.out.q : p.out.k) + img * (PK * IMG);
    for (int i = tid * 16; i < PK * IMG; i += 256 * 16) *(u32x4*)(to + i) = *(const u32x4*)(lds + which * PK * IMG + i);
  }

  // ---- K K^T and Q K^T, row tile `wave`, column tiles up to it: lane has column 16 jt + r, rows 4 gq + e
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) kk[jt] = qk[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < DKB; ++s) {
    const f16x8 ka = rows_frag<DKP>(lds, wave, s, r, gq), qa = rows_frag<DKP>(lds + PK * IMG, wave, s, r, gq);
    f16x8 kal, qal;
    if constexpr (PK == 2) {
      kal = rows_frag<DKP>(lds + IMG, wave, s, r, gq);
      qal = rows_frag<DKP>(lds + 3 * IMG, wave, s, r, gq);
    }
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      if (jt > wave) continue;
      const f16x8 kb = rows_frag<DKP>(lds, jt, s, r, gq);
      if constexpr (PK == 2) {
        const f16x8 kbl = rows_frag<DKP>(lds + IMG, jt, s, r, gq);
        kk[jt] = mfma(kal, kb, kk[jt]);
        kk[jt] = mfma(ka, kbl, kk[jt]);
        qk[jt] = mfma(qal, kb, qk[jt]);
        qk[jt] = mfma(qa, kbl, qk[jt]);
      }
      kk[jt] = mfma(ka, kb, kk[jt]);
      qk[jt] = mfma(qa, kb, qk[jt]);
    }
  }
  __syncthreads();  // the images' place is A, T and P from here

  for (int rep = 0; rep < group; ++rep) {
    const int h = hk * group + rep;
    const int64_t bh = (int64_t)b * p.NH + h, part = bh * p.chunks + chunk;
    // ---- running sums of g, a lane a token
    if (rep) load_gates(bh);
    gt = gt < CLAMP_G ? CLAMP_G : gt;
    double sum = (double)gt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double below = __shfl_up(sum, o, 64);
      if (lane >= o) sum += below;
    }
    const double last = __shfl(sum, 63, 64);
    if (wave == 0) {
      bs[lane] = sum;
      betas[lane] = bt;
      Factors* f = p.out.f + part;
      const float in = exp_of(sum), ks = ksc[lane], qs = qsc[lane];
      f->b[lane] = sum;
      f->in[lane] = in * ks;
      f->q[lane] = in * qs * p.scale;
      f->out[lane] = exp_of(last - sum) * ks;
      f->back[lane] = bt * in * ks;
      f->k[lane] = exponent_of(ks);
      f->qs[lane] = exponent_of(qs);
      f->beta[lane] = bt;
    }
    __syncthreads();
    // ---- A and P
    double bi[4];
    float be[4], sp[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * wave + 4 * gq + e;
      bi[e] = bs[i];
      be[e] = betas[i] * ksc[i];
      sp[e] = p.scale * qsc[i];
    }
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      const int j = 16 * jt + r;
      const double bj = bs[j];
      const float kj = BWD || betas[j] != 0.f ? ksc[j] : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * wave + 4 * gq + e;
        const float dec = jt <= wave && j <= i ? exp_of(bi[e] - bj) * kj : 0.f;
        Am[i * MLD + j] = j < i ? be[e] * dec * kk[jt][e] : 0.f;
        Pm[i * MLD + j] = j <= i ? sp[e] * dec * qk[jt][e] : 0.f;
        Tm[i * MLD + j] = 0.f;
      }
    }
    __syncthreads();
    // ---- the diagonal blocks' inverses: lane r has column r
    {
      const float* a = Am + 16 * wave * MLD + 16 * wave;
      float t[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x = i == r ? 1.f : 0.f;
#pragma unroll
        for (int l = 0; l < i; ++l) x = fmaf(-a[i * MLD + l], t[l], x);
        t[i] = x;
      }
      if (lane < 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) Tm[(16 * wave + i) * MLD + 16 * wave + r] = t[i];
      }
    }
    __syncthreads();
    // ---- block column `wave`, downwards
    f32x4 col[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) col[0][e] = Tm[(16 * wave + 4 * gq + e) * MLD + 16 * wave + r];
#pragma unroll
    for (int d = 1; d < 4; ++d) {  // block row wave + d
      if (wave + d > 3) continue;
      const int i = wave + d;
      f32x4 m = {0.f, 0.f, 0.f, 0.f}, n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int l = 0; l < d; ++l) {
        const f32x4 a = *(const f32x4*)(Am + (16 * i + r) * MLD + 16 * (wave + l) + 4 * gq);
#pragma unroll
        for (int e = 0; e < 4; ++e) m = mfma4(a[e], col[l][e], m);
      }
      const f32x4 a = *(const f32x4*)(Tm + (16 * i + r) * MLD + 16 * i + 4 * gq);
#pragma unroll
      for (int e = 0; e < 4; ++e) n = mfma4(a[e], m[e], n);
      col[d] = -n;
    }
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      if (wave + d > 3) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) Tm[(16 * (wave + d) + 4 * gq + e) * MLD + 16 * wave + r] = col[d][e];
    }
    __syncthreads();
    // ---- operands: wave w has the 16 rows 16 w .. of each matrix, both halves of k
    constexpr int FORMS = BWD ? 2 : 1;  // P, T; P^T, T^T
    Factors* f = p.out.f + part;
    const int i = 16 * wave + r;
    auto column = [&](int half, int e) { return 32 * half + (e < 4 ? 4 * gq + e : 12 + 4 * gq + e); };
    auto write = [&](f16_t* to, const float (&x)[2][8], float up, bool with_lo) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f16x8 hi, lo;
        split8<true>(x[half], up, hi, lo);
        f16_t* at = to + part * (2 * FRAG_PLANE) + ((2 * wave + half) * 64 + lane) * 8;
        *(f16x8*)at = hi;
        if (with_lo) *(f16x8*)(at + FRAG_PLANE) = lo;
      }
    };
#pragma unroll
    for (int turned = 0; turned < FORMS; ++turned) {  // P: a scale a row
      float x[2][8], m = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = column(half, e);
          x[half][e] = turned ? Pm[j * MLD + i] : Pm[i * MLD + j];
          m = fmaxf(m, fabsf(x[half][e]));
        }
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const Pow2 sc = pow2_for(m, 10);
      write(turned ? p.out.pt : p.out.p, x, sc.up, BWD || !std::is_same_v<T, bf16_t>);  // bf16's scan takes P as one plane
      if (gq == 0) {
        if (turned) f->pt[i] = sc.down;
        else f->p[i] = exponent_of(sc.down);
      }
    }
    float x[FORMS][2][8], m[FORMS];
#pragma unroll
    for (int turned = 0; turned < FORMS; ++turned) {  // T: one scale
      m[turned] = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = column(half, e);
          x[turned][half][e] = turned ? Tm[j * MLD + i] : BWD && betas[j] == 0.f ? 0.f : Tm[i * MLD + j];
          m[turned] = fmaxf(m[turned], fabsf(x[turned][half][e]));
        }
    }
    block_max(m, red);
#pragma unroll
    for (int turned = 0; turned < FORMS; ++turned) write(turned ? p.out.tt : p.out.t, x[turned], pow2_for(m[turned], 10).up, true);
    if (tid == 0) {
      f->all = exp_of(last);
      f->t = pow2_for(m[0], 10).down;
      f->tt = BWD ? pow2_for(m[FORMS - 1], 10).down : 0.f;
    }
    __syncthreads();
  }
}

template <typename T, bool BWD>
const void* pick(int dkp) {
  return dkp == 64 ? (const void*)delta_prep_kernel<T, 2, BWD> : dkp == 128 ? (const void*)delta_prep_kernel<T, 4, BWD>
                                                                           : (const void*)delta_prep_kernel<T, 8, BWD>;
}

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

}  // namespace

size_t prep_bytes(const Shape& s, bool backward) {
  const int64_t frags = up256(s.parts() * 2 * FRAG_PLANE * 2);
  return 2 * up256(s.images() * s.image_bytes()) + (backward ? 4 : 2) * frags + up256(s.parts() * (int64_t)sizeof(Factors));
}

Prep prep_at(const Shape& s, bool backward, char* ws) {
  const int64_t image = up256(s.images() * s.image_bytes()), frags = up256(s.parts() * 2 * FRAG_PLANE * 2);
  Prep p{};
  p.k = ws;
  p.q = p.k + image;
  char* at = p.q + image;
  p.t = (f16_t*)at;
  p.p = (f16_t*)(at + frags);
  if (backward) {
    p.tt = (f16_t*)(at + 2 * frags);
    p.pt = (f16_t*)(at + 3 * frags);
  }
  p.f = (Factors*)(at + (backward ? 4 : 2) * frags);
  return p;
}

int launch_prep(const Shape& s, const void* q, const void* k, const void* g, const void* beta, const Prep& out, bool backward,
                hipStream_t st, const char* who) {
  PrepArgs a{q, k, g, beta, {}, {}, s.NH, s.NHK, s.S, s.DK, s.chunks(), s.scale, s.dtype_gates, false, out};
  int64_t any = 0;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = s.qs[i];
    a.ks[i] = s.ks[i];
    any |= s.qs[i] | s.ks[i];
  }
  a.wide = any % (16 / dtype_size(s.dtype)) == 0 && (((uintptr_t)q | (uintptr_t)k) & 15) == 0;
  const void* kern = s.dtype == XL_DTYPE_F32    ? backward ? pick<float, true>(s.dkp()) : pick<float, false>(s.dkp())
                     : s.dtype == XL_DTYPE_BF16 ? backward ? pick<bf16_t, true>(s.dkp()) : pick<bf16_t, false>(s.dkp())
                                                : backward ? pick<f16_t, true>(s.dkp()) : pick<f16_t, false>(s.dkp());
  int64_t lds = 2 * s.image_bytes();
  if (lds < 3 * L * MLD * 4) lds = 3 * L * MLD * 4;
  void* args[] = {&a};
  hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e == hipSuccess) e = hipLaunchKernel(kern, dim3((unsigned)s.images()), dim3(256), args, (unsigned)lds, st);
  if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
  return check_launch(who);
}

}  // namespace delta
}  // namespace xl
