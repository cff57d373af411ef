// Gated linear unit of a feed-forward block and its gradients:
//
//   a = x Wg^T,  u = x Wu^T,  h = act(a) u          x [T, D], Wg, Wu [F, D]
//   da = dh u act'(a),  du = dh act(a),  dx = da Wg + du Wu,  dWg = da^T x,  dWu = du^T x
//
// The forward is one product of x with both weights: a tile holds the same rows of Wg and of Wu, a wave has a and u of the
// same values in its registers, and only h goes to memory (for training a and u too, in float32: the gradients' factors
// keep their bits).  Backward: da and du once, zero-padded to whole slices; dx as one product over both weights' rows; the
// weights' gradients as one launch of two; both in parts of K where tiles are few.  Up to 16 tokens the weights are streamed
// past them instead.
//
// Products: 16 x 16 blocks of v_mfma_f32_16x16x32, sums in registers; slices of 64 of K of both operands in LDS, STAGES of
// them, filled straight from memory STAGES - 1 ahead; a wave holds the operands of 32 of a slice's 64 and multiplies them
// while it reads those of the next 32; one barrier a slice.  An operand whose K is contiguous lies by rows [row][8 pieces of
// 16 bytes], piece p at p ^ (row % 8); one whose K is the row index by columns [k][pieces of 32 bytes], read by LDS reads
// that transpose.  The loads write LDS in lane order, so each lane fetches what belongs at its place.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "mfma_bf16.h"

namespace xl {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

enum Act { SILU = 0, GELU = 1 };
enum Product { FWD, DX, DW };  // h; dx; dWg and dWu
enum Part { WHOLE, PART, JOIN };  // a tile; a part of its sum over K; the tile from its parts, added in order

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same_v<T, bf16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 16 bytes from float32, two values by one conversion
template <typename T>
__device__ __forceinline__ T rounded1(float v) {
  using pair = std::conditional_t<std::is_same_v<T, f16_t>, xl_f16x2, xl_bf16x2>;
  const uint16_t x = (uint16_t)__builtin_bit_cast(uint32_t, __builtin_convertvector((xl_f32x2{v, 0.f}), pair));
  return __builtin_bit_cast(T, x);
}
template <typename T>
__device__ __forceinline__ u32x4 rounded8(const float (&v)[8]) {
  using pair = std::conditional_t<std::is_same_v<T, f16_t>, xl_f16x2, xl_bf16x2>;
  u32x4 raw;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    raw[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((xl_f32x2{v[2 * j], v[2 * j + 1]}), pair));
  return raw;
}

// act(a) and its derivative; exp by the hardware's exp2, a few units of float32 off, far below a 16-bit result's rounding.  GELU by erfc:
// 1 + erf cancels below zero (at a = -4 to 11 bits).
__device__ __forceinline__ float act_of(float a, int act) {
  if (act == SILU) return a * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(a * -1.4426950408889634f));
  return 0.5f * a * erfcf(a * -0.70710678118654752f);
}
__device__ __forceinline__ float act_grad(float a, int act, float& value) {
  if (act == SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(a * -1.4426950408889634f));
    value = a * s;
    return s * fmaf(a, 1.f - s, 1.f);
  }
  const float phi = 0.5f * erfcf(a * -0.70710678118654752f);
  value = a * phi;
  return fmaf(a * 0.3989422804014327f, __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f), phi);
}

// 16 bytes a lane from global memory into LDS, at lds + 16 * lane (lds the same in the whole wave).  Written out, so that
// the compiler does not wait for it before the next LDS read; m0 has to be written one wait state before the load.  Whoever
// reads what it writes waits for it by vmcnt, and then for everybody at a barrier.
__device__ __forceinline__ void to_lds(uint32_t lds, uint32_t offset, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void to_lds(uint32_t lds, const void* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory");
}
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ const u32x4 glu_zeros = {0u, 0u, 0u, 0u};

// sum[l][r] over k of left[l][k] right[r][k]; out [r][l]
struct Args {
  // FWD: left Wg, Wu [F, K], right x [T, K].  DX: left Wg, Wu [K, D] by columns, right da, du [T, K], one after the other.
  // DW: left x [K, D] by columns, right da, du [K, F] by columns, each for itself.
  const void *left[2], *right[2];
  int64_t left_pitch, right_pitch;  // elements, multiples of 8
  int lefts, rights, K;             // FWD: lefts F; K (for DX of one weight; multiples of 64 are read, see below)
  int left_rows;                    // rows of an operand by columns: past them the last is read again, against zeros
  int left_tiles, right_tiles;
  void* out[2];
  int64_t out_pitch;
  float *a, *u;  // FWD: a, u [T, keep_pitch], or null
  int64_t keep_pitch;
  int act;
  bool wide;  // rows of out are multiples of 8 values
  int splits;      // parts of K
  float* partial;  // their sums, by [tile][part]
};

template <int BL, int BR, int WL, int WR, int STAGES, int MODE, int PARTS, typename T>
__global__ __launch_bounds__(64 * WL * WR) void glu_product_kernel(Args p) {
  constexpr int THREADS = 64 * WL * WR, BK = 64, TL = BL / WL / 16, TR = BR / WR / 16;
  constexpr bool LC = MODE != FWD, RC = MODE == DW;  // by columns
  constexpr int STAGE = (BL + BR) * 128;
  constexpr int PER = THREADS / 8;                                       // rows of 128 bytes by one load of the workgroup
  constexpr int LK = THREADS * 8 / BL, RK = THREADS * 8 / BR;            // rows k of BL or BR columns by one
  constexpr int LOADS_L = BL / PER, LOADS = LOADS_L + BR / PER, READS = TL + TR;
  static_assert(BL % PER == 0 && BR % PER == 0 && (!LC || LK % 16 == 0) && (!RC || RK % 16 == 0) && LOADS * (STAGES - 2) < 64);
  static_assert(MODE != FWD || TL % 2 == 0);
  extern __shared__ __align__(1024) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wl = wave / WR, wr = wave % WR;

  // neighbours share operands, on one XCD
  const int tiles = p.left_tiles * p.right_tiles, job = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int all = PARTS == PART ? __builtin_amdgcn_readfirstlane(job / p.splits) : job, split = PARTS == PART ? job - all * p.splits : 0;
  const int b = __builtin_amdgcn_readfirstlane(all / tiles), t = all - b * tiles;
  constexpr int G = 4;
  const int group = t / (G * p.left_tiles), rows = min(G, p.right_tiles - group * G), in = t - group * G * p.left_tiles;
  const int br = __builtin_amdgcn_readfirstlane(group * G + in % rows), bl = __builtin_amdgcn_readfirstlane(in / rows);

  // where this lane's loads come from: byte offsets from the operands' slices
  const int64_t ll = p.left_pitch * 2, lr = p.right_pitch * 2;
  const int piece = ((tid & 7) ^ ((tid >> 3) & 7)) * 16;
  // 64 columns: a row is half the banks, so rows of one parity need the keys
  auto key_of = [](int wide, int k) { return wide >= 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2); };
  // a column operand's load: row k of the slice's first rows, byte offset of its 8 columns
  auto column_of = [&](int wide, int first, int count, int& k) {
    const int pieces = wide / 8, at = tid % pieces;
    k = tid / pieces;
    return min(first + ((((at >> 1) ^ key_of(wide, k)) << 1) | (at & 1)) * 8, count - 8) * 2;
  };
  int lk = 0, rk = 0;
  uint32_t from_l[LC ? 1 : LOADS_L], from_r[RC ? 1 : LOADS - LOADS_L];
  // FWD: a wave's rows of the tile are as many of Wg, then the same of Wu; the 8 rows that a wave loads are of one of them
  constexpr int HALF = BL / WL / 2, FS = BL / 2;
  bool up_l[LOADS_L];
  const int l_cols = MODE == FWD ? 0 : (p.lefts + 7) / 8 * 8, r_cols = RC ? (p.rights + 7) / 8 * 8 : 0;
  if constexpr (LC) {
    const int column = column_of(BL, bl * BL, l_cols, lk);
    from_l[0] = (uint32_t)(lk * ll + column);
  } else {
#pragma unroll
    for (int i = 0; i < LOADS_L; ++i) {
      const int row = i * PER + (tid >> 3), w = row / (2 * HALF), r = row % (2 * HALF);
      up_l[i] = __builtin_amdgcn_readfirstlane(r / HALF) != 0;
      from_l[i] = (uint32_t)(min(w * HALF + r % HALF, p.lefts - 1 - bl * FS) * ll + piece);
    }
  }
  if constexpr (RC) {
    const int column = column_of(BR, br * BR, r_cols, rk);
    from_r[0] = (uint32_t)(rk * lr + column);
  } else {
#pragma unroll
    for (int i = 0; i < BR / PER; ++i)
      from_r[i] = (uint32_t)(min(i * PER + (tid >> 3), p.rights - 1 - br * BR) * lr + piece);
  }
  const int per_weight = (p.K + BK - 1) / BK, whole = MODE == DX ? 2 * per_weight : per_weight;
  const int first = PARTS == PART ? __builtin_amdgcn_readfirstlane((int)((int64_t)whole * split / p.splits)) : 0;
  const int slices = PARTS == PART ? __builtin_amdgcn_readfirstlane((int)((int64_t)whole * (split + 1) / p.splits)) : whole;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_char*)lds + wave * 1024;
  auto fetch_one = [&](auto I, int slice, int stage) {
    constexpr int i = I.value;
    const uint32_t to = lds_at + stage * STAGE + i * (PER * 128);
    const int which = MODE == DX ? slice >= per_weight : MODE == DW ? b : 0, k = MODE == DX && which ? slice - per_weight : slice;
    const int64_t k0 = (int64_t)k * BK;
    if constexpr (i < LOADS_L) {
      if constexpr (LC) {
        const char* base = (const char*)p.left[MODE == DX ? which : 0] + (k0 + i * LK) * ll;
        const int left = p.left_rows - 1 - (int)k0 - i * LK;  // rows that are there past the first
        if (left >= LK - 1)
          to_lds(to, from_l[0], base);
        else  // 32 rows at most, back from the first
          to_lds(to, base + min(lk, left) * ll + (from_l[0] - (uint32_t)(lk * ll)));
      } else {
        const char* base = (const char*)p.left[up_l[i] ? 1 : 0] + bl * FS * ll + k0 * 2;
        if (k0 + BK <= p.K)
          to_lds(to, from_l[i], base);
        else
          to_lds(to, k0 + piece / 2 < p.K ? base + from_l[i] : (const char*)&glu_zeros);
      }
    } else if constexpr (RC) {
      to_lds(to, from_r[0], (const char*)p.right[which] + (k0 + (i - LOADS_L) * RK) * lr);
    } else {
      const char* base = (const char*)p.right[MODE == DX ? which : 0] + br * BR * lr + k0 * 2;
      if (MODE == DX || k0 + BK <= p.K)
        to_lds(to, from_r[i - LOADS_L], base);
      else
        to_lds(to, k0 + piece / 2 < p.K ? base + from_r[i - LOADS_L] : (const char*)&glu_zeros);
    }
  };

  f32x4 acc[TL][TR];
#pragma unroll
  for (int i = 0; i < TL; ++i)
#pragma unroll
    for (int j = 0; j < TR; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int row = lane & 15, quad = lane >> 4;
  struct Half {  // a wave's operands of 32 of a slice's 64
    u32x4 l[TL], r[TR];
  };
  const int by_row = row * 128 + ((quad ^ (row & 7)) << 4), first_k = quad * 8 + (row >> 2);
  const int by_column_l = first_k * (BL * 2) + (key_of(BL, first_k) ^ (wl * TL)) * 32 + (row & 3) * 8;
  const int by_column_r = first_k * (BR * 2) + (key_of(BR, first_k) ^ (wr * TR)) * 32 + (row & 3) * 8;
  // read I of half s of the slice at LDS offset `base`: 8 values along k, from 32 s + 8 quad, of a row or a column
  auto read_one = [&](auto I, Half& h, int base, int s) {
    constexpr int i = I.value;
    const char* at = lds + base;
    if constexpr (i < TL) {
      if constexpr (LC) {
        at += s * (32 * BL * 2) + (by_column_l ^ (i * 32));
        h.l[i] = __builtin_bit_cast(u32x4, mfma::tr_pair(at, at + 4 * BL * 2));
      } else {
        h.l[i] = *(const u32x4*)(at + (wl * TL + i) * 2048 + (by_row ^ (s * 64)));
      }
    } else if constexpr (RC) {
      at += BL * 128 + s * (32 * BR * 2) + (by_column_r ^ ((i - TL) * 32));
      h.r[i - TL] = __builtin_bit_cast(u32x4, mfma::tr_pair(at, at + 4 * BR * 2));
    } else {
      h.r[i - TL] = *(const u32x4*)(at + BL * 128 + (wr * TR + i - TL) * 2048 + (by_row ^ (s * 64)));
    }
  };
  // one half's products, a row of blocks at a time, each with its share of the next half's reads and of `more`
  auto multiply = [&](const Half& h, Half& next, int next_base, int next_s, auto&& more) {
    mfma::static_for<0, TL>([&](auto I) {
      constexpr int i = I.value;
      mfma::static_for<READS * i / TL, READS * (i + 1) / TL>([&](auto R) { read_one(R, next, next_base, next_s); });
      more(I);
#pragma unroll
      for (int j = 0; j < TR; ++j) acc[i][j] = mfma16<T>(h.l[i], h.r[j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // all but this wave's last LEFT loads are in LDS, and its reads done; then everybody's
  auto landed = [&](auto LEFT) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT.value) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Past the end the last slice is loaded again, and read, but not multiplied: the same number of loads is under way after
  // every slice.
  using Behind = std::integral_constant<int, LOADS*(STAGES - 2)>;
  // a lane's sums of a part: one f32x4 a block, the workgroup's side by side
  auto part_at = [&](int of, int at) { return (f32x4*)p.partial + (((int64_t)all * p.splits + of) * (TL * TR) + at) * THREADS + tid; };
  if constexpr (PARTS == JOIN) {
    for (int of = 0; of < p.splits; ++of)
#pragma unroll
      for (int i = 0; i < TL; ++i)
#pragma unroll
        for (int j = 0; j < TR; ++j) acc[i][j] += *part_at(of, i * TR + j);
  } else {
    Half h0, h1;
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k)
      mfma::static_for<0, LOADS>([&](auto I) { fetch_one(I, min(first + k, slices - 1), k); });
    landed(Behind{});
    mfma::static_for<0, READS>([&](auto R) { read_one(R, h0, 0, 0); });
    mfma::static_for<0, LOADS>([&](auto I) { fetch_one(I, min(first + STAGES - 1, slices - 1), STAGES - 1); });
    int stage = 0;
    for (int k = first; k < slices; ++k) {
      const int next = stage + 1 == STAGES ? 0 : stage + 1, ahead = min(k + STAGES, slices - 1);
      multiply(h0, h1, stage * STAGE, 1, [](auto) {});
      landed(Behind{});  // slice k + 1 is there, slice k has been read
      multiply(h1, h0, next * STAGE, 0, [&](auto I) {
        mfma::static_for<LOADS * I.value / TL, LOADS * (I.value + 1) / TL>([&](auto X) { fetch_one(X, ahead, stage); });
      });
      stage = next;
    }
    landed(std::integral_constant<int, 0>{});
  }
  if constexpr (PARTS == PART) {
#pragma unroll
    for (int i = 0; i < TL; ++i)
#pragma unroll
      for (int j = 0; j < TR; ++j) *part_at(split, i * TR + j) = acc[i][j];
    return;
  }

  // A lane has left 4 quad .. 4 quad + 3 of right `row` of each block: 16 rows at a time, turned in the wave's own part of LDS
  constexpr int OUT = MODE == FWD ? TL / 2 : TL, LDW = OUT * 16 + 4, EACH = OUT * 2;
  float* strip = (float*)lds + wave * (16 * LDW);
  const int l0 = MODE == FWD ? bl * FS + wl * HALF : bl * BL + wl * TL * 16, r0 = br * BR + wr * TR * 16;
  T* out = (T*)p.out[MODE == DW ? b : 0];
#pragma unroll
  for (int j = 0; j < TR; ++j) {
    wave_fence();
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
      f32x4 v = acc[i][j];
      if constexpr (MODE == FWD) {
        const f32x4 u = acc[TL / 2 + i][j];
        const int f = l0 + i * 16 + quad * 4, tok = r0 + j * 16 + row;
        if (p.a && tok < p.rights && f < p.lefts) {  // keep_pitch is a multiple of 4
          *(f32x4*)(p.a + tok * p.keep_pitch + f) = v;
          *(f32x4*)(p.u + tok * p.keep_pitch + f) = u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = act_of(v[e], p.act) * u[e];
      }
      *(f32x4*)(strip + row * LDW + i * 16 + quad * 4) = v;
    }
    wave_fence();
    if (p.wide) {
#pragma unroll
      for (int h = 0; h < (16 * EACH + 63) / 64; ++h) {
        const int at = h * 64 + lane, r = at / EACH, c = at % EACH * 8, m = r0 + j * 16 + r, n = l0 + c;
        if (r >= 16 || m >= p.rights || n >= p.lefts) continue;
        const f32x4 v0 = *(const f32x4*)(strip + r * LDW + c), v1 = *(const f32x4*)(strip + r * LDW + c + 4);
        const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        *(u32x4*)(out + m * p.out_pitch + n) = rounded8<T>(v);
      }
    } else {  // rows of any address: neighbouring lanes write neighbouring values
#pragma unroll 4
      for (int h = 0; h < 4 * OUT; ++h) {
        const int at = h * 64 + lane, r = at / (OUT * 16), c = at % (OUT * 16), m = r0 + j * 16 + r, n = l0 + c;
        if (m < p.rights && n < p.lefts) out[m * p.out_pitch + n] = rounded1<T>(strip[r * LDW + c]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ few tokens
// 16 rows of Wg and of Wu a workgroup, its waves share K; the parts meet in LDS.  Tokens past T read the last one again.  Bound by
// memory: 8 tokens of 4096 to 10944 43 us, 4.2 TB/s.  Waves and 32s of K that each has under way, us for those 8 tokens, 8 of 2048 to
// 5504 and 4 of 8192 to 1024: 8 and 2 43.2, 15.9, 23.8; 8 and 4 45.2, 17.8, 25.4; 4 and 2 42.0, 14.9, 27.4; 4 and 8 42.7, 16.5, 29.6;
// 16 and 2 43.6, 17.3, 24.4; 8 and 1 49.4, 17.4, 25.5.
constexpr int FEW_WAVES = 8, FEW_KB = 2, FEW_TOKENS = 16;

template <typename T>
__global__ __launch_bounds__(64 * FEW_WAVES) void glu_few_kernel(const T* __restrict__ x, const T* __restrict__ wg,
                                                                 const T* __restrict__ wu, T* __restrict__ h, int M, int D,
                                                                 int F, int act) {
  __shared__ f32x4 parts[FEW_WAVES - 1][2][64];
  const int lane = threadIdx.x & 63, g = lane >> 4, r16 = lane & 15, wv = threadIdx.x >> 6;
  const int f0 = blockIdx.x * 16, nk = (D + 31) / 32, nkw = (nk + FEW_WAVES - 1) / FEW_WAVES;
  const int kbeg = wv * nkw, kend = min(nk, kbeg + nkw);
  const size_t wrow = (size_t)min(f0 + r16, F - 1) * D + 8 * g;
  const T *gr = wg + wrow, *ur = wu + wrow, *xr = x + (size_t)min(r16, M - 1) * D + 8 * g;
  // k-slice [32 ks + 8 g, +8) lies wholly inside or outside D; outside, the address is clamped and the operands are zeros
  auto koff = [&](int ks) { return min(32 * ks, D - 8 - 8 * g); };
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, u = a;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int k0 = kbeg; k0 < kend; k0 += FEW_KB) {
    u32x4 wa[FEW_KB], wb[FEW_KB], xb[FEW_KB];
#pragma unroll
    for (int p = 0; p < FEW_KB; ++p) {
      const int ko = koff(min(k0 + p, nk - 1));
      wa[p] = __builtin_nontemporal_load((const u32x4*)(gr + ko));
      wb[p] = __builtin_nontemporal_load((const u32x4*)(ur + ko));
      xb[p] = *(const u32x4*)(xr + ko);
    }
#pragma unroll
    for (int p = 0; p < FEW_KB; ++p) {
      const bool in = k0 + p < kend && 32 * (k0 + p) + 8 * g < D;
      const u32x4 b = in ? xb[p] : zero;
      a = mfma16<T>(in ? wa[p] : zero, b, a);
      u = mfma16<T>(in ? wb[p] : zero, b, u);
    }
  }
  if (wv > 0) {
    parts[wv - 1][0][lane] = a;
    parts[wv - 1][1][lane] = u;
  }
  __syncthreads();
  if (wv > 0 || r16 >= M) return;
#pragma unroll
  for (int q = 0; q < FEW_WAVES - 1; ++q) {
    a += parts[q][0][lane];
    u += parts[q][1][lane];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int f = f0 + 4 * g + e;
    if (f < F) h[(size_t)r16 * F + f] = from_f32<T>(act_of(a[e], act) * u[e]);
  }
}

// ------------------------------------------------------------------------------------------------ da, du
// [Tp, Fp], zero past T and F; 8 values a thread.  Rounded once, to the type, for the matrix cores, as a block of two 16-bit projections rounds
// them too: the weights' gradients have two roundings, and float16's da and du end at 65504 and 2^-25, as dh does.
template <typename T>
__global__ __launch_bounds__(256) void glu_factors_kernel(const T* __restrict__ dh, const float* __restrict__ a,
                                                          const float* __restrict__ u, int64_t keep_pitch, T* __restrict__ da,
                                                          T* __restrict__ du, int tokens, int F, int Fp, int64_t pieces, int act,
                                                          bool wide) {
  const int per = Fp / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per;
    const int f = (int)(i - t * per) * 8;
    float ga[8], gu[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) ga[e] = gu[e] = 0.f;
    if (t < tokens && f < F) {
      float d[8];
      if (wide && f + 8 <= F) {
        struct alignas(16) Eight { T e[8]; };
        const Eight v = *(const Eight*)(dh + t * F + f);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = to_f32(v.e[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = f + e < F ? to_f32(dh[t * F + f + e]) : 0.f;
      }
      const f32x4 *ap = (const f32x4*)(a + t * keep_pitch + f), *up = (const f32x4*)(u + t * keep_pitch + f);
      const f32x4 av[2] = {ap[0], ap[1]}, uv[2] = {up[0], up[1]};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float value;
        const float slope = act_grad(av[e >> 2][e & 3], act, value);
        ga[e] = f + e < F ? d[e] * (uv[e >> 2][e & 3] * slope) : 0.f;
        gu[e] = f + e < F ? d[e] * value : 0.f;
      }
    }
    *(u32x4*)(da + i * 8) = rounded8<T>(ga);
    *(u32x4*)(du + i * 8) = rounded8<T>(gu);
  }
}

// rows [R, C] to [R, Cp], zeros past C: for rows that 16 bytes do not fit
template <typename T>
__global__ __launch_bounds__(256) void glu_pad_kernel(const T* __restrict__ from, T* __restrict__ to, int C, int Cp, int64_t count) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / Cp;
    const int c = (int)(i - r * Cp);
    to[i] = c < C ? from[r * C + c] : from_f32<T>(0.f);
  }
}

// ------------------------------------------------------------------------------------------------ host
constexpr int CUS = 256;
int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

unsigned grid_of(int64_t count) {
  const int64_t n = (count + 255) / 256;
  return (unsigned)(n < 16384 ? n : 16384);
}

template <int BL, int BR, int WL, int WR, int STAGES, int MODE, int PARTS, typename T>
int launch_part(const Args& a, const char* who, hipStream_t st) {
  constexpr int TL = BL / WL / 16, OUT = MODE == FWD ? TL / 2 : TL;
  constexpr int STRIPS = WL * WR * 16 * (OUT * 16 + 4) * 4, SLICES = PARTS == JOIN ? 0 : STAGES * (BL + BR) * 128;
  constexpr int LDS = SLICES > STRIPS ? SLICES : STRIPS;
  static_assert(LDS <= 160 * 1024);
  auto kernel = glu_product_kernel<BL, BR, WL, WR, STAGES, MODE, PARTS, T>;
  if (LDS > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  }
  const int64_t tiles = (int64_t)a.left_tiles * a.right_tiles * (MODE == DW ? 2 : 1) * (PARTS == PART ? a.splits : 1);
  if (tiles > 0x7fffffff) return set_error(XL_ERR_UNSUPPORTED, "%s: too many tiles", who);
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * WL * WR), LDS, st, a);
  return check_launch(who);
}

// Tiles: the cheapest by the rounds of the chip that they take, us a slice of K and round, and what a round costs besides (its first
// loads, its end).  Measured, whole products in us: 777 tokens of 2048 to 5504, h: 256 x 192 46, 256 x 256 53, 128 x 128 63, 64 x 64
// 75; 1333 of 1000 to 2731: 128 x 128 29, 256 x 192 32, 256 x 256 37; 300 of 1024 to 2752: 64 x 64 10, 128 x 128 14; 128 of 4096 to
// 10944: 128 x 128 in four stages 43, in two 57, 64 x 64 47; 8192 of those: 256 x 256 1127, 256 x 192 1239, 128 x 128 1512.  (256 x 128,
// 128 x 256, 128 x 64 and 256 x 64 were nowhere better by more than 10 %.)
enum Tile { T256, T192, T128_2, T128_4, T64, TILES };
struct Shape {
  int bl, br;
  double slice, round;
};
constexpr Shape SHAPES[TILES] = {{256, 256, 1.6, 5.0}, {256, 192, 1.28, 4.5}, {128, 128, 0.57, 2.5}, {128, 128, 0.52, 3.0}, {64, 64, 0.215, 2.0}};

// A product's tile and the parts of its K.  A sum over many slices of few tiles is split, its parts kept in float32 and joined by a
// second launch: 4 us, what it writes and reads, and 25 bytes a ns that one workgroup reads.  Measured with da and du, us: dx of 777
// tokens of 2048 to 5504 87 whole, 72 in two parts of 128 x 128; of 128 tokens of 4096 to 10944 101 and 54; of 64 of 2048 to 5504 57 and
// 21.  h has two sums a tile and long K only with many tiles: whole.
struct Plan {
  int tile = T64, splits = 1;
  int64_t tiles = 0;
  size_t partial() const { return splits > 1 ? (size_t)tiles * splits * SHAPES[tile].bl * SHAPES[tile].br * 4 : 0; }
};
Plan plan(int mode, int64_t lefts, int64_t rights, int64_t K) {
  const int64_t whole = (K + 63) / 64 * (mode == DX ? 2 : 1);
  Plan best;
  double least = INFINITY;
  for (int tile = 0; tile < TILES; ++tile) {
    if (tile == T192 && mode != FWD) continue;
    const Shape& s = SHAPES[tile];
    const int64_t l = mode == FWD ? s.bl / 2 : s.bl, tiles = (lefts + l - 1) / l * ((rights + s.br - 1) / s.br) * (mode == DW ? 2 : 1);
    for (int splits = 1; splits <= (mode == FWD ? 1 : 8); ++splits) {
      if (splits > 1 && whole < 8 * splits) break;
      const int64_t rounds = (tiles * splits + CUS - 1) / CUS, slices = (whole + splits - 1) / splits;
      if (tile == T128_4 && rounds > 1) continue;
      double us = rounds * (slices * s.slice + s.round);
      if (tile == T128_2 && rounds == 1) us += slices * 0.1;
      if (splits > 1) us += 4.0 + std::max((double)tiles * splits * s.bl * s.br * 8 / 4.5e6, (double)splits * s.bl * s.br * 4 / 25e3);
      if (us < least) {
        least = us;
        best.tile = tile;
        best.splits = splits;
        best.tiles = tiles;
      }
    }
  }
  return best;
}

template <int BL, int BR, int WL, int WR, int STAGES, int MODE, typename T>
int launch_tiles(Args a, const char* who, hipStream_t st) {
  constexpr int LEFT = MODE == FWD ? BL / 2 : BL;
  a.left_tiles = (a.lefts + LEFT - 1) / LEFT;
  a.right_tiles = (a.rights + BR - 1) / BR;
  if constexpr (MODE != FWD) {
    if (a.splits > 1) {
      const int rc = launch_part<BL, BR, WL, WR, STAGES, MODE, PART, T>(a, who, st);
      return rc ? rc : launch_part<BL, BR, WL, WR, STAGES, MODE, JOIN, T>(a, who, st);
    }
  }
  return launch_part<BL, BR, WL, WR, STAGES, MODE, WHOLE, T>(a, who, st);
}

template <int MODE, typename T>
int launch_product(Args a, char* partial, const char* who, hipStream_t st) {
  const Plan use = plan(MODE, a.lefts, a.rights, a.K);
  a.splits = use.splits;
  a.partial = (float*)partial;
  if (use.tile == T256) return launch_tiles<256, 256, 2, 4, 2, MODE, T>(a, who, st);
  if constexpr (MODE == FWD)
    if (use.tile == T192) return launch_tiles<256, 192, 2, 4, 2, MODE, T>(a, who, st);
  if (use.tile == T128_2) return launch_tiles<128, 128, 2, 2, 2, MODE, T>(a, who, st);
  if (use.tile == T128_4) return launch_tiles<128, 128, 2, 2, 4, MODE, T>(a, who, st);
  return launch_tiles<64, 64, 2, 2, 4, MODE, T>(a, who, st);
}

// What both directions need in workspace: x and the weights by rows of whole 16 bytes, where D is not a multiple of 8; the
// backward da and du besides, and the sums of a product's parts (dx's, then the weights').
struct Layout {
  int64_t Dp, Fp, Tp, x, w, factor, partial = 0;
  Layout(int64_t tokens, int D, int F, bool backward) {
    const bool pad = D % 8 != 0 && (backward || tokens > 0);
    Dp = up_to(D, 8);
    Fp = up_to(F, 64);
    Tp = up_to(tokens, 64);
    x = pad ? up_to(tokens * Dp * 2, 256) : 0;
    w = pad ? up_to((int64_t)F * Dp * 2, 256) : 0;
    factor = backward ? up_to(Tp * Fp * 2, 256) : 0;
    if (backward && tokens > 0) {
      const size_t dx = plan(DX, D, tokens, Fp).partial(), dw = plan(DW, D, F, Tp).partial();
      partial = (int64_t)(dx > dw ? dx : dw);
    }
  }
  int64_t bytes() const { return x + 2 * w + 2 * factor + partial; }
};

int check_sizes(const char* who, int64_t tokens, int D, int F, int act, int dtype) {
  if (tokens < 0 || D < 1 || F < 1) return set_error(XL_ERR_INVALID_ARG, "%s: negative tokens, or D or F below 1", who);
  if (!dtype_ok(dtype)) return set_error(XL_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
  if (act != SILU && act != GELU) return set_error(XL_ERR_INVALID_ARG, "%s: unknown activation %d", who, act);
  if (dtype == XL_DTYPE_F32) return set_error(XL_ERR_UNSUPPORTED, "%s: float32 (bfloat16 and float16 only)", who);
  // 256 rows of an operand are within 32-bit byte offsets
  if (tokens > (1 << 28) || D > (1 << 22) || F > (1 << 22)) return set_error(XL_ERR_UNSUPPORTED, "%s: sizes too large", who);
  return XL_OK;
}

template <typename T>
const void* padded(const void* from, char* to, int64_t rows, int D, int Dp, hipStream_t st) {
  const int64_t count = rows * Dp;
  glu_pad_kernel<T><<<grid_of(count), 256, 0, st>>>((const T*)from, (T*)to, D, Dp, count);
  return to;
}

template <typename T>
int forward(const void* x, const void* wg, const void* wu, void* h, float* a, float* u, int64_t keep_pitch, int tokens, int D,
            int F, int act, const Layout& lay, char* ws, hipStream_t st, const char* who) {
  if (!a && tokens <= FEW_TOKENS && D % 8 == 0) {
    glu_few_kernel<T><<<(F + 15) / 16, 64 * FEW_WAVES, 0, st>>>((const T*)x, (const T*)wg, (const T*)wu, (T*)h, tokens, D, F, act);
    return check_launch(who);
  }
  if (lay.x) {
    x = padded<T>(x, ws, tokens, D, (int)lay.Dp, st);
    wg = padded<T>(wg, ws + lay.x, F, D, (int)lay.Dp, st);
    wu = padded<T>(wu, ws + lay.x + lay.w, F, D, (int)lay.Dp, st);
  }
  Args p{};
  p.left[0] = wg;
  p.left[1] = wu;
  p.right[0] = x;
  p.left_pitch = p.right_pitch = lay.Dp;
  p.lefts = F;
  p.rights = tokens;
  p.K = (int)lay.Dp;
  p.out[0] = h;
  p.out_pitch = F;
  p.a = a;
  p.u = u;
  p.keep_pitch = keep_pitch;
  p.act = act;
  p.wide = F % 8 == 0;
  return launch_product<FWD, T>(p, nullptr, who, st);
}

template <typename T>
int backward(const void* dh, const void* x, const void* wg, const void* wu, const float* a, const float* u, int64_t keep_pitch,
             void* dx, void* dwg, void* dwu, int tokens, int D, int F, int act, const Layout& lay, char* ws, hipStream_t st,
             const char* who) {
  if (lay.x) {
    if (dwg) x = padded<T>(x, ws, tokens, D, (int)lay.Dp, st);
    if (dx) {
      wg = padded<T>(wg, ws + lay.x, F, D, (int)lay.Dp, st);
      wu = padded<T>(wu, ws + lay.x + lay.w, F, D, (int)lay.Dp, st);
    }
  }
  T *da = (T*)(ws + lay.x + 2 * lay.w), *du = (T*)((char*)da + lay.factor);
  char* const partial = (char*)du + lay.factor;
  const int64_t pieces = lay.Tp * (lay.Fp / 8);
  glu_factors_kernel<T><<<grid_of(pieces), 256, 0, st>>>((const T*)dh, a, u, keep_pitch, da, du, tokens, F, (int)lay.Fp, pieces, act,
                                                       F % 8 == 0);
  if (const int rc = check_launch(who)) return rc;
  if (dx) {
    Args p{};
    p.left[0] = wg;
    p.left[1] = wu;
    p.right[0] = da;
    p.right[1] = du;
    p.left_pitch = lay.Dp;
    p.right_pitch = lay.Fp;
    p.lefts = D;
    p.rights = tokens;
    p.K = (int)lay.Fp;
    p.left_rows = F;
    p.out[0] = dx;
    p.out_pitch = D;
    p.wide = D % 8 == 0;
    if (const int rc = launch_product<DX, T>(p, partial, who, st)) return rc;
  }
  if (dwg) {
    Args p{};
    p.left[0] = x;
    p.right[0] = da;
    p.right[1] = du;
    p.left_pitch = lay.Dp;
    p.right_pitch = lay.Fp;
    p.lefts = D;
    p.rights = F;
    p.K = (int)lay.Tp;
    p.left_rows = tokens;
    p.out[0] = dwg;
    p.out[1] = dwu;
    p.out_pitch = D;
    p.wide = D % 8 == 0;
    if (const int rc = launch_product<DW, T>(p, partial, who, st)) return rc;
  }
  return XL_OK;
}

}  // namespace
}  // namespace xl

extern "C" size_t xl_gated_linear_workspace_size(int64_t T, int D, int F, int backward, int dtype) {
  using namespace xl;
  if (check_sizes("xl_gated_linear_workspace_size", T, D, F, 0, dtype) != XL_OK) return 0;
  return (size_t)Layout(T, D, F, backward != 0).bytes();
}

extern "C" int xl_gated_linear_fwd(const void* x, const void* w_gate, const void* w_up, void* h, float* a, float* u,
                                   int64_t keep_pitch, int64_t T, int D, int F, int act, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace xl;
  const char* who = "xl_gated_linear_fwd";
  clear_error();
  if (const int rc = check_sizes(who, T, D, F, act, dtype)) return rc;
  if (T == 0) return XL_OK;
  if (!x || !w_gate || !w_up || !h) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if ((a == nullptr) != (u == nullptr)) return set_error(XL_ERR_INVALID_ARG, "%s: a and u go together", who);
  if (a && (keep_pitch < F || keep_pitch % 8)) return set_error(XL_ERR_INVALID_ARG, "%s: keep_pitch must be a multiple of 8, at least F", who);
  if (((uintptr_t)x | (uintptr_t)w_gate | (uintptr_t)w_up | (uintptr_t)h | (uintptr_t)a | (uintptr_t)u) & 15)
    return set_error(XL_ERR_INVALID_ARG, "%s: pointers must be 16-byte aligned", who);
  const Layout lay(T, D, F, false);
  if (lay.bytes() && (!workspace || workspace_bytes < (size_t)lay.bytes() || ((uintptr_t)workspace & 255)))
    return set_error(XL_ERR_WORKSPACE, "%s: the workspace must be %zu bytes, 256-byte aligned", who, (size_t)lay.bytes());
  if (dtype == XL_DTYPE_BF16)
    return forward<bf16_t>(x, w_gate, w_up, h, a, u, keep_pitch, (int)T, D, F, act, lay, (char*)workspace, (hipStream_t)stream, who);
  return forward<f16_t>(x, w_gate, w_up, h, a, u, keep_pitch, (int)T, D, F, act, lay, (char*)workspace, (hipStream_t)stream, who);
}

extern "C" int xl_gated_linear_bwd(const void* dh, const void* x, const void* w_gate, const void* w_up, const float* a,
                                   const float* u, int64_t keep_pitch, void* dx, void* dw_gate, void* dw_up, int64_t T, int D,
                                   int F, int act, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace xl;
  const char* who = "xl_gated_linear_bwd";
  clear_error();
  if (const int rc = check_sizes(who, T, D, F, act, dtype)) return rc;
  if ((dw_gate == nullptr) != (dw_up == nullptr)) return set_error(XL_ERR_INVALID_ARG, "%s: dw_gate and dw_up go together", who);
  if (!dx && !dw_gate) return XL_OK;
  if (T == 0) return set_error(XL_ERR_INVALID_ARG, "%s: no tokens", who);
  if (!dh || !x || !w_gate || !w_up || !a || !u) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (keep_pitch < F || keep_pitch % 8) return set_error(XL_ERR_INVALID_ARG, "%s: keep_pitch must be a multiple of 8, at least F", who);
  if (((uintptr_t)dh | (uintptr_t)x | (uintptr_t)w_gate | (uintptr_t)w_up | (uintptr_t)a | (uintptr_t)u | (uintptr_t)dx |
       (uintptr_t)dw_gate | (uintptr_t)dw_up) & 15)
    return set_error(XL_ERR_INVALID_ARG, "%s: pointers must be 16-byte aligned", who);
  const Layout lay(T, D, F, true);
  if (!workspace || workspace_bytes < (size_t)lay.bytes() || ((uintptr_t)workspace & 255))
    return set_error(XL_ERR_WORKSPACE, "%s: the workspace must be %zu bytes, 256-byte aligned", who, (size_t)lay.bytes());
  if (dtype == XL_DTYPE_BF16)
    return backward<bf16_t>(dh, x, w_gate, w_up, a, u, keep_pitch, dx, dw_gate, dw_up, (int)T, D, F, act, lay, (char*)workspace,
                            (hipStream_t)stream, who);
  return backward<f16_t>(dh, x, w_gate, w_up, a, u, keep_pitch, dx, dw_gate, dw_up, (int)T, D, F, act, lay, (char*)workspace,
                         (hipStream_t)stream, who);
}
