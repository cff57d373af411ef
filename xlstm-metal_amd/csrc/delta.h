// The gated delta rule by chunks of 64 tokens: what its kernels share (chunkwise forward: delta_chunkwise.hip, backward:
// delta_backward.hip).
//
//   S_t = a_t S_{t-1} + k_t d_t^T,  d_t = beta_t (v_t - (a_t S_{t-1})^T k_t),  h_t = scale S_t^T q_t,  a_t = exp(g_t)
//
// In a chunk, with b_i = g_1 + .. + g_i, c_i = exp(b_i), D_ij = exp(b_i - b_j) and S the state before it (rows i, j are tokens):
//
//   A_ij = beta_i D_ij k_i.k_j (j < i),  T = (I + A)^-1,  U = T R,  R = diag(beta) (V - diag(c) K S),  P_ij = scale D_ij q_i.k_j (j <= i)
//   H = scale diag(c) Q S + P U,   S' = c_L S + (diag(c_L / c_j) K)^T U
//
// T and P do not know the state: a first kernel (delta_prep) forms them for all chunks at once.  What is left of a chunk
// acts on each column of V, U and S by itself: a scan takes blocks of 16 columns through the whole sequence, a block's [DQK, 16]
// piece of the state in float32 registers, and no block waits for another.
//
// All products are on the matrix cores in f16 with float32 sums.  Every operand stands at a power-of-two scale that puts its
// largest value high in f16's range: each row of K, of Q and of P at its own, so that a token's h has its bits beside tokens of other
// sizes; T at a chunk's; S, R and U at a block of columns'.  Largest values from 2^-86 to 2^110 are kept.  float32 values enter
// as pairs hi + lo of f16 (22 bits), and a product of two pairs is three.  f16 ends at 2^-24: a value x times below its operand's largest is
// off by 2^-25 of that where this stands at 1 (K, Q), by 2^-39 where at 2^14 (R, U), if that is more than 2^-22 (one plane: 2^-11) of itself.
//
// Operand layout of v_mfma_f32_16x16x32_f16: lane l = 16 g + r holds row (A) or column (B) r, k = 8 g .. 8 g + 7; the result's
// column is r, its rows 4 g .. 4 g + 3.  Two results below each other (16 rows each) hold 4 g + e and 16 + 4 g + e of 32 rows:
// they are the next product's B operand as they stand if its A operand has k in that order.  "Turned" 32s have it: piece g
// of 8 values holds 4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3.
#pragma once

#include <stddef.h>

#include "common.h"
#include "mfma_bf16.h"

namespace xl {
namespace delta {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int L = 64;           // tokens of a chunk
// f16 planes of K and Q: pairs for float32; 16-bit values have their bits in one
template <typename T>
constexpr int PLANES = is_f32<T>::value ? 2 : 1;
// Planes that the backward keeps of U, Z, dH and the states (KEPT, 0 in the forward): pairs, but one where inputs and gates are bf16, whose own
// rounding is 8 times a plane's.  The gates' gradients are made of differences that show it: one plane takes a float32 dg 3e-5 to
// 6e-4 of its terms off, pairs below 1e-5.
inline int kept_planes(int dtype, int dtype_gates) { return dtype == XL_DTYPE_BF16 && dtype_gates == XL_DTYPE_BF16 ? 1 : 2; }
constexpr int MAX_DQK = 256;
constexpr int FRAGS = 8;        // 16 x 32 operands of a 64 x 64 matrix: row tile mt, half s of k at 2 mt + s
constexpr int FRAG_PLANE = FRAGS * 64 * 8;  // f16 values of one plane
constexpr float CLAMP_G = -1e4f;  // exp() of it is 0: a reset (-inf) keeps the sums finite

// Per head and chunk, by the first kernel: per-token factors (the scales of K's and Q's rows, 2^k_i and 2^q_i, folded in) and scales, the bytes
// as biased exponents.  A row of zeros has scale 0.
struct Factors {
  float back[L];    // beta_i c_i 2^k_i    K S; Z into the state's gradient
  float q[L];       // scale c_i 2^q_i     Q S
  float out[L];     // c_L / c_i 2^k_i     U into the state
  float beta[L];    // the scan by several waves takes this 1 KB into LDS, and what follows to P's rows into registers,
  float all, t;     // c_L; T = planes * t
  uint8_t p[L];     // P's rows = planes * these
  float tt;         // T^T
  float pad[45];    // that by one wave 1.25 KB,
  float pt[L];      // P^T's rows
  float in[L];      // c_i 2^k_i
  uint8_t k[L], qs[L];  // K's and Q's rows
  float pad2[32];   // the scan backwards 2 KB
  double b[L];      // running sums of g
};
static_assert(sizeof(Factors) == 2560 && offsetof(Factors, all) == 1024 && offsetof(Factors, b) == 2048);
__device__ __forceinline__ float power_of(uint32_t exponent) { return __uint_as_float(exponent << 23); }
__device__ __forceinline__ uint8_t exponent_of(float power) { return (uint8_t)(__float_as_uint(power) >> 23); }

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A barrier for what lies in LDS; loads from memory stay under way (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Every load and store under way, also to the compiler, which counts what it knows of
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// the scheduler's order here: N products, a few vector operations between them
template <int N>
__device__ __forceinline__ void interleave() {
  mfma::static_for<0, N>([](auto) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
  });
}

// 2^target / 2^exponent(m) and its inverse: m times the first is in [2^target, 2^(target + 1)); m >= 0.
// At most 2^100 either way (0 gets that).
struct Pow2 {
  float up, down;
};
__device__ __forceinline__ Pow2 pow2_for(float m, int target = 14) {
  const int e = (int)(__float_as_uint(m) >> 23);
  int sh = e == 255 ? 0 : target + 127 - e;
  sh = sh > 100 ? 100 : sh < -100 ? -100 : sh;
  return {__uint_as_float((uint32_t)(127 + sh) << 23), __uint_as_float((uint32_t)(127 - sh) << 23)};
}

// exp(x): float32's rounding of x alone would cost |x| 2^-24 of the result
__device__ __forceinline__ float exp_of(double x) {
  const float hi = (float)x, e = expf(hi);
  return fmaf(e, (float)(x - (double)hi), e);
}

// max over the wave of x >= 0, in every lane (scalar); by the bits, which order as the values do.  A lane's infinity or NaN does not count: a
// lane has values of one column, and its neighbours keep their scale.
__device__ __forceinline__ float wave_max_all(float value) {
  uint32_t x = __float_as_uint(value);
  x = x < 0x7f800000u ? x : 0u;
#define XL_DPP_MAX(CTRL, ROWMASK) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWMASK, 0xf, false));
  XL_DPP_MAX(0x111, 0xf)  // row_shr:1 (what is shifted in is 0)
  XL_DPP_MAX(0x112, 0xf)
  XL_DPP_MAX(0x114, 0xf)
  XL_DPP_MAX(0x118, 0xf)
  XL_DPP_MAX(0x142, 0xa)  // row_bcast:15
  XL_DPP_MAX(0x143, 0xc)  // row_bcast:31
#undef XL_DPP_MAX
  return __int_as_float(__builtin_amdgcn_readlane((int)x, 63));
}

__device__ __forceinline__ uint32_t pk_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((xl_f32x2{a, b}), xl_f16x2));
}
// x as f16 planes, 8 values, x within f16's range
__device__ __forceinline__ void split8(f32x4 x, f32x4 y, f16x8& hi, f16x8& lo) {
  u32x4 h, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = j < 2 ? x[2 * j] : y[2 * j - 4], b = j < 2 ? x[2 * j + 1] : y[2 * j - 3];
    const xl_f16x2 p = __builtin_convertvector((xl_f32x2{a, b}), xl_f16x2);
    h[j] = __builtin_bit_cast(uint32_t, p);
    l[j] = pk_f16(a - (float)p[0], b - (float)p[1]);
  }
  hi = __builtin_bit_cast(f16x8, h);
  lo = __builtin_bit_cast(f16x8, l);
}
// x * scale as planes, 4 values
__device__ __forceinline__ void split4(f32x4 x, float scale, f16x4& hi, f16x4& lo) {
  u32x2 h, l;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float a = x[2 * j], b = x[2 * j + 1];
    const xl_f16x2 p = __builtin_convertvector((xl_f32x2{a * scale, b * scale}), xl_f16x2);
    h[j] = __builtin_bit_cast(uint32_t, p);
    l[j] = pk_f16(fmaf(a, scale, -(float)p[0]), fmaf(b, scale, -(float)p[1]));
  }
  hi = __builtin_bit_cast(f16x4, h);
  lo = __builtin_bit_cast(f16x4, l);
}
__device__ __forceinline__ f16x8 join(f16x4 a, f16x4 b) {
  return f16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// a / b of powers of two, as f16 (0 below its range); a <= b
__device__ __forceinline__ _Float16 ratio(float a, float b) {
  const int e = (int)(__float_as_uint(a) >> 23) - (int)(__float_as_uint(b) >> 23);
  return e < -24 ? (_Float16)0.f : (_Float16)__uint_as_float((uint32_t)(127 + e) << 23);
}
// x * scale as f16 planes, 8 values
template <bool PAIR>
__device__ __forceinline__ void split8(const float (&x)[8], float scale, f16x8& hi, f16x8& lo) {
  u32x4 h, l = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = x[2 * j], b = x[2 * j + 1];
    const xl_f16x2 p = __builtin_convertvector((xl_f32x2{a * scale, b * scale}), xl_f16x2);
    h[j] = __builtin_bit_cast(uint32_t, p);
    if constexpr (PAIR) l[j] = pk_f16(fmaf(a, scale, -(float)p[0]), fmaf(b, scale, -(float)p[1]));
  }
  hi = __builtin_bit_cast(f16x8, h);
  lo = __builtin_bit_cast(f16x8, l);
}
// 16 bytes at a uniform base and a lane's 32-bit offset
__device__ __forceinline__ f16x8 load16(const void* base, uint32_t at) { return *(const f16x8*)((const char*)base + at); }
// 4 neighbours, rounded
template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T e[4];
};
template <typename T>
__device__ __forceinline__ Four<T> rounded4(f32x4 v) {
  if constexpr (is_f32<T>::value) {
    return __builtin_bit_cast(Four<T>, v);
  } else {
    using pair = std::conditional_t<std::is_same_v<T, f16_t>, xl_f16x2, xl_bf16x2>;
    return __builtin_bit_cast(Four<T>, (u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector((xl_f32x2{v[0], v[1]}), pair)),
                                             __builtin_bit_cast(uint32_t, __builtin_convertvector((xl_f32x2{v[2], v[3]}), pair))}));
  }
}
template <bool PAIR>
__device__ __forceinline__ void split8(f32x4 a, f32x4 b, float scale, f16x8& hi, f16x8& lo) {
  const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  split8<PAIR>(x, scale, hi, lo);
}

// 16 bytes a lane from global memory into LDS, at lds + 16 * lane (lds the same in the whole wave).  Whoever reads what it
// writes waits for it by vmcnt, and then for everybody at a barrier.  m0 has to be written one wait state before.
__device__ __forceinline__ void to_lds(uint32_t lds, uint32_t offset, const void* base) {
  // a base that the compiler has moved to vector registers comes back
  base = (const void*)((uint64_t)(uint32_t)uniform((int)((uint64_t)base >> 32)) << 32 | (uint32_t)uniform((int)(uint64_t)base));
  lds = (uint32_t)uniform((int)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}

// The scans keep the state at a power-of-two scale: its planes are taken without a multiplication.  With max(c_L |S|, |w|)
// below 2^(STATE + 1) and K's values below 2 the next state, c_L S + K^T w over 64 tokens, is below 129 2^(STATE + 1) = 33024.
// A chunk's products are summed from zero and added to the state once: in the matrix cores' sums every one of them would
// round the state, towards zero.
constexpr int STATE = 7;
constexpr int STATE_BACK = 6;  // two products: 257 2^7 = 32896

__device__ __forceinline__ f32x4 fma4(f32x4 x, float a, f32x4 y) {
  return f32x4{fmaf(x[0], a, y[0]), fmaf(x[1], a, y[1]), fmaf(x[2], a, y[2]), fmaf(x[3], a, y[3])};
}
// max of |x| of a lane's
template <int N>
__device__ __forceinline__ float abs_max(const f32x4 (&x)[N]) {
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], fabsf(x[t][e]));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// max of |x| over a wave's piece of the state
template <int N>
__device__ __forceinline__ float state_max(const f32x4 (&st)[N]) {
  return wave_max_all(abs_max(st));
}

// Images of K and Q: [plane][64 tokens][DKP] f16, each token's largest value in [1, 2), each 32 columns turned, the 16-byte piece p
// of token i at p ^ (i % 8).
template <int DKP>
__device__ __forceinline__ int piece_at(int token, int p) {
  return token * (DKP * 2) + ((p ^ (token & 7)) << 4);
}
// A or B operand: tokens 16 mt .. + 15, columns of half s (32 s ..), as turned
template <int DKP>
__device__ __forceinline__ f16x8 rows_frag(const char* img, int mt, int s, int r, int g) {
  return *(const f16x8*)(img + piece_at<DKP>(16 * mt + r, 4 * s + g));
}
// A operand: columns 16 t .. + 15 (one a lane), k = tokens 32 s + (4 g .. , 16 + 4 g ..)
template <int DKP>
__device__ __forceinline__ f16x8 columns_frag(const char* img, int t, int s, int r, int g) {
  const int token = 32 * s + 4 * g + (r >> 2), p = 4 * (t >> 1) + (r & 3);
  const char* a = img + piece_at<DKP>(token, p) + (t & 1) * 8;
  return __builtin_bit_cast(f16x8, mfma::tr_pair(a, a + 16 * DKP * 2));  // 16 tokens on: the same token % 8
}

// The operands of a 64 x 64 matrix with nothing above its diagonal (below, for a transposed one): 6 of the 8.
constexpr int LOWER = 6;
__device__ __host__ constexpr int lower_mt(int i) { return i < 2 ? i : 2 + (i - 2) / 2; }
__device__ __host__ constexpr int lower_s(int i) { return i < 2 ? 0 : (i - 2) % 2; }
__device__ __forceinline__ void load_lower(const f16_t* from, uint32_t lane, f16x8 (&to)[LOWER]) {
#pragma unroll
  for (int i = 0; i < LOWER; ++i) to[i] = load16(from + (2 * lower_mt(i) + lower_s(i)) * 512, lane * 16);
}
// of a transposed one: row tiles 0 and 1 have both halves of k, 2 and 3 the second
__device__ __host__ constexpr int upper_mt(int i) { return i < 4 ? i / 2 : i - 2; }
__device__ __host__ constexpr int upper_s(int i) { return i < 4 ? i % 2 : 1; }
__device__ __forceinline__ void load_upper(const f16_t* from, uint32_t lane, f16x8 (&to)[LOWER]) {
#pragma unroll
  for (int i = 0; i < LOWER; ++i) to[i] = load16(from + (2 * upper_mt(i) + upper_s(i)) * 512, lane * 16);
}

// What the backward keeps of a scan for the chunks' gradients, by 16 columns n (a wave's): tokens x n, [plane][16 n][64 tokens,
// turned], and states, [plane][16 n][DKP, turned], f16 at a scale of their own.  Blocks of 16 are padded to an even number.
struct Kept {
  f16_t *u, *z, *dh;   // tokens x n
  f16_t *s0, *ds;      // the state before the chunk, the gradient of the state behind it
  float *us, *zs, *dhs, *s0s, *dss;  // values = planes * these, powers of two (a block of zeros: the least)
  int blocks;          // of a head, padded
};
__device__ __forceinline__ int64_t kept_at(int64_t part, int blocks, int block, int planes, int width) {
  return ((part * blocks + block) * planes) * (int64_t)(16 * width);
}

// ------------------------------------------------------------------------------------------------ workspace, shapes
struct Shape {
  int B, NH, NHK, S, DK, DV;
  int64_t qs[3], ks[3], vs[3];  // element strides of batch, head, token
  float scale;
  int dtype, dtype_gates;
  int chunks() const { return (S + L - 1) / L; }
  int dkp() const { return DK <= 64 ? 64 : DK <= 128 ? 128 : 256; }
  int kept() const { return kept_planes(dtype, dtype_gates); }
  int64_t images() const { return (int64_t)B * NHK * chunks(); }
  int64_t parts() const { return (int64_t)B * NH * chunks(); }
  int64_t image_bytes() const { return (int64_t)(dtype == XL_DTYPE_F32 ? 2 : 1) * L * dkp() * 2; }
};

// What the first kernel writes; transposed forms for the backward only.
struct Prep {
  char *k, *q;       // images
  f16_t *t, *p;      // [part][plane][FRAG_PLANE]: T (2 planes), P; columns of tokens of beta 0: delta_prep.hip
  f16_t *tt, *pt;    // T^T, P^T (2 planes)
  Factors* f;
};

int check_shape(const char* who, const Shape& s);
// q, k, v strides from the caller's nine or of contiguous tensors
int set_strides(Shape& s, const int64_t* strides, const char* who);
constexpr int MAX_TOKEN_STRIDE = 1 << 22;
size_t prep_bytes(const Shape& s, bool backward);
Prep prep_at(const Shape& s, bool backward, char* ws);
int launch_prep(const Shape& s, const void* q, const void* k, const void* g, const void* beta, const Prep& p, bool backward,
                hipStream_t st, const char* who);
// The scan: h (and c_last), or for the backward every chunk's U and state before it.
int launch_scan(const Shape& s, const void* v, const float* c0, void* h, float* c_last, const Prep& prep, const Kept* kept,
                hipStream_t st, const char* who);
int launch_recurrent(const Shape& s, const void* q, const void* k, const void* v, const void* g, const void* beta,
                     const float* c0, void* h, float* c_last, hipStream_t st, const char* who);

}  // namespace delta
}  // namespace xl
