// Orthogonalisation of a matrix by Newton-Schulz products:
//
//   X = G / (|G|_F + eps);  steps times:  A = X X^T,  P = b A + c A^2,  X = a X + P X
//
// on the side with fewer rows (G^T for a tall G), so that every singular value s goes to s (a + b s^2 + c s^4) a step.
// The products are on the matrix cores in f16 with float32 sums.  Every matrix is kept at a power-of-two scale that
// holds it in f16's range.  For f16 and float32 every matrix is a pair hi + lo of f16 (22 bits) and a product three (hi hi
// + hi lo + lo hi): 1.7e-6 of the norm at 1777 x 1000, where float32 products lose 2.6e-6.  For bf16, which enters
// exactly, one f16 plane is enough for a few steps: five of Muon's end 1.7e-3 to 2.1e-3 of the norm off for spread
// singular values (the result's own rounding: 1.65e-3; bf16 intermediates: 1e-2 to 3e-2), up to 5.3e-3 for a matrix of
// low rank, up to 1e-2 where rows repeat and their roundings add up.  P's diagonal, its largest values, stays in float32
// beside it and joins a (2.35e-3 with it in f16).  What is rounded away in the directions of small singular values
// grows with them, so bf16 with coefficients that let it grow further runs pairs too: see MOST_NOISE.
//
// A and P are symmetric: their tiles on and below the diagonal are computed and written to both places.  X is kept
// by rows; P X reads it down its columns with LDS reads that transpose.  All matrices are zero-padded to multiples of
// 64 in the workspace, and a tile past the end reads its last rows again: no bounds in the loops, and products of
// zeros stay zero.
//
// Large matrices are bound by the matrix cores (4096 x 4096 bf16: P X 111 us, 1240 TFLOP/s, where a library f16 product
// takes 109) and, in the symmetric products' smaller tiles, by LDS reads; middling ones in batches by memory (12 of
// 1024 x 2048: P X 70 us, 300 MB); small ones by latency and launches.  us for five steps, by machine: 4096 x 4096 1280
// to 1410, 10944 x 4096 2860 to 3100, 12 of 1024 x 2048 660 to 740, 1777 x 1000 float32 217 to 223, 128 x 128 28 (the
// products with torch in float32: 14400, 32050, 5550, 627, 492); 4096 x 4096 float32 3940 to 4110, float16 3890 to 4000,
// 128 x 128 float16 48.
#include <math.h>

#include <type_traits>

#include "common.h"
#include "mfma_bf16.h"

namespace xl {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
template <typename T>
using raw_at = std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4>;
template <typename T>
struct Vec {  // 16 bytes, at any element's address
  T e[16 / sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  const u32x4 raw = *(const raw_at<T>*)p;
  return __builtin_bit_cast(Vec<T>, raw);
}
// 16 bytes of T from float32, two values by one conversion
template <typename T>
__device__ __forceinline__ u32x4 rounded_vec(const float* v) {
  if constexpr (is_f32<T>::value) {
    return __builtin_bit_cast(u32x4, (f32x4{v[0], v[1], v[2], v[3]}));
  } else {
    using pair = std::conditional_t<std::is_same_v<T, f16_t>, xl_f16x2, xl_bf16x2>;
    u32x4 raw;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      raw[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((xl_f32x2{v[2 * j], v[2 * j + 1]}), pair));
    return raw;
  }
}
template <typename T>
struct Four {
  T e[4];
};
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
template <typename T>
using raw_four = std::conditional_t<sizeof(T) == 2, u32x2_at2, u32x4_at4>;
template <typename T>
__device__ __forceinline__ Four<T> load_four(const T* p) {
  const std::conditional_t<sizeof(T) == 2, u32x2, u32x4> raw = *(const raw_four<T>*)p;
  return __builtin_bit_cast(Four<T>, raw);
}
template <typename T>
__device__ __forceinline__ void store_four(T* p, const Four<T>& v) {
  *(raw_four<T>*)p = __builtin_bit_cast(std::conditional_t<sizeof(T) == 2, u32x2, u32x4>, v);
}
typedef __attribute__((address_space(3))) char lds_char;

// stored = value * scale: with |singular values| of X up to 8 (checked on the host), |A| <= 64 and |P| <= 250.  X is scaled
// up further where it cannot grow that large (factors_of).
constexpr float SCALE_X = 256.f, SCALE_A = 256.f, SCALE_P = 64.f;
constexpr float MOST_X = 8.f, MOST_P = 250.f;
// The most that the roundings of all steps may have grown to, in units of one step's, for products of single planes: each
// step multiplies what is there by at most its polynomial's largest slope.  Five of Muon's steps: 489; six: 2157; twelve of
// (1.5, -0.5, 0): 257.  Errors relative to the norm, bf16 matrices of exactly rank 8 or 32, single planes and pairs:
// five steps 4.3e-3 and 1.7e-3, six 1.4e-2 and 1.7e-3, eight 0.16 and 2.0e-3, ten 1.8 and 1.3e-2 (float32 products, rounded:
// ten 2.0e-2).  us, six steps: 4096 x 4096 1570 and 4940, 12 of 1024 x 2048 836 and 1950, 128 x 128 32 and 58.
constexpr double MOST_NOISE = 512.0;

// ------------------------------------------------------------------------------------------------ norm and first X
constexpr int NORM_BLOCK = 512, NORM_PARTS = 256;  // most partial sums of a matrix

template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void ns_norm_kernel(const T* __restrict__ g, int64_t count, int parts,
                                                             double* __restrict__ part) {
  constexpr int VW = 16 / sizeof(T), AHEAD = 4;
  __shared__ double sums[NORM_BLOCK / 64];
  const T* p = g + blockIdx.y * count;
  const int64_t whole = count / VW, step = (int64_t)parts * NORM_BLOCK, at = (int64_t)blockIdx.x * NORM_BLOCK + threadIdx.x;
  double s = 0.0;  // no float32 value's square overflows it
  auto add = [&](float f) {
    const double v = (double)f;
    s = fma(v, v, s);
  };
  int64_t i = at;
  for (; i + (AHEAD - 1) * step < whole; i += AHEAD * step) {
    Vec<T> v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) v[u] = load_vec(p + (i + u * step) * VW);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int j = 0; j < VW; ++j) add(to_f32(v[u].e[j]));
  }
  for (; i < whole; i += step) {
    const Vec<T> v = load_vec(p + i * VW);
#pragma unroll
    for (int j = 0; j < VW; ++j) add(to_f32(v.e[j]));
  }
  if (at < count - whole * VW) add(to_f32(p[whole * VW + at]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.0;
#pragma unroll
  for (int w = 0; w < NORM_BLOCK / 64; ++w) s += sums[w];
  part[(int64_t)blockIdx.y * parts + blockIdx.x] = s;
}

constexpr int MOST_STEPS = 64;
struct Coefficients {  // a kernel's argument
  float v[3 * MOST_STEPS];
};

// A matrix's factors: X0 = stored * first, later X = stored * later.
struct Factors {
  float first, later;
};
__device__ __forceinline__ Factors factors_of(double norm, double eps, double growth, double& enter) {
  int e = 0;
  enter = 1.0;
  if (norm > 0.0 && norm < 1.7e308) {
    frexp(norm, &e);
    enter = ldexp(1.0, 13 - e);  // |stored|_F in [2^12, 2^13)
  }
  // A G far below eps keeps its smallness: it is scaled up by what the steps cannot make up for, to singular values of up
  // to 128 (2^15 as stored), so that the lo planes keep their bits.  (Up to 1, 4096 x 4096 float32 of a hundredth of eps and
  // below were up to 8e-5 off.)
  int up = 0;
  const double share = norm / (norm + eps) * growth / 128.0;
  if (share > 0.0 && share < 1.0) {
    frexp(share, &up);
    up = up < -110 ? 110 : up < 0 ? -up : 0;
  }
  // zeros stay zeros however small eps is: the square of 1 / eps would not be finite
  const double first = norm == 0.0 && eps > 0.0 ? 0.0 : 1.0 / ((norm + eps) * enter);
  return Factors{(float)first, (float)ldexp(1.0 / SCALE_X, -up)};
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

__device__ __forceinline__ void store_planes(f16_t* to, int64_t lo_plane, bool with_lo, const float (&v)[8]) {
  f16x8 hi, lo;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    _Float16 h, l;
    split(v[q], h, l);
    hi[q] = h;
    lo[q] = l;
  }
  *(f16x8*)to = hi;
  if (with_lo) *(f16x8*)(to + lo_plane) = lo;
}

// X [Mp, Np] (f16 planes, zero past the matrix) from G [M, N], or from G [N, M] (TALL); 64 x 64 a workgroup
template <typename T, int PL, bool TALL>
__global__ __launch_bounds__(256) void ns_enter_kernel(const T* __restrict__ g, int M, int N, int Mp, int Np,
                                                       const double* __restrict__ part, int parts, double eps,
                                                       double growth, f16_t* __restrict__ x, int64_t x_plane,
                                                       Factors* __restrict__ factors) {
  constexpr int VW = 16 / sizeof(T);
  __shared__ float tile[TALL ? 64 : 1][65];
  __shared__ double sums[4], scale;
  const int tid = threadIdx.x, b = blockIdx.z;
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, R = TALL ? N : M, C = TALL ? M : N;
  const int r0 = TALL ? n0 : m0, c0 = TALL ? m0 : n0;
  const T* gp = g + (int64_t)b * M * N;
  f16_t* xp = x + (int64_t)b * Mp * Np;
  const int r = tid >> 3, c = (tid & 7) * 8;  // 8 values of rows r and r + 32, of G's tile and of X's
  float v[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int rr = r0 + r + 32 * h;
    const T* from = gp + (int64_t)rr * C + c0 + c;
    if (rr < R && c0 + c + 8 <= C) {
#pragma unroll
      for (int q = 0; q < 8; q += VW) {
        const Vec<T> u = load_vec(from + q);
#pragma unroll
        for (int j = 0; j < VW; ++j) v[h][q + j] = to_f32(u.e[j]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[h][q] = rr < R && c0 + c + q < C ? to_f32(from[q]) : 0.f;
    }
  }
  double s = tid < parts ? part[(int64_t)b * parts + tid] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((tid & 63) == 0) sums[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    double enter;
    const Factors f = factors_of(sqrt(sums[0] + sums[1] + sums[2] + sums[3]), eps, growth, enter);
    if (blockIdx.x == 0 && blockIdx.y == 0) factors[b] = f;
    scale = enter;
  }
  __syncthreads();
  const double enter = scale;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int q = 0; q < 8; ++q) v[h][q] = (float)((double)v[h][q] * enter);
  if constexpr (TALL) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 8; ++q) tile[r + 32 * h][c + q] = v[h][q];
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 8; ++q) v[h][q] = tile[c + q][r + 32 * h];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
    store_planes(xp + (int64_t)(m0 + r + 32 * h) * Np + n0 + c, x_plane, PL == 2, v[h]);
}

// ------------------------------------------------------------------------------------------------ the products
// 16 bytes a lane from global memory into LDS, at lds + 16 * lane (lds the same in the whole wave).  Written out, so that
// the compiler does not wait for it before the next LDS read; nothing else here uses m0, which has to be written one
// wait state before the load.  Whoever reads what it writes waits for it by vmcnt, and then for everybody at a barrier.
__device__ __forceinline__ void to_lds(uint32_t lds, uint32_t offset, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

enum Product { XXT, XXT_PART, XXT_JOIN, AA, PX, LAST };  // A, a part of its sums, A from the parts; P; X; the result

// sum[l][r] over k of left[l][k] right[r][k]
struct Args {
  // left [lefts, K] by rows (A, X), or X [K, lefts] by columns (PX, LAST); right [rights, K]; planes hi, and lo a plane on
  const f16_t *left, *right;
  int64_t left_plane, right_plane, left_batch, right_batch;
  int lefts, rights, K;     // multiples of 64
  int left_tiles, right_tiles;
  // XXT_PART, XXT_JOIN: parts of K, their sums by [tile][split]
  int splits;
  float* partial;
  // value = beta * e + alpha * sum; e as out
  const f16_t* e;
  int64_t e_plane, e_batch;
  int e_planes;
  float alpha, beta;
  float* diagonal;  // one plane: P's [batch, Mp], at P's scale; AA writes it and zeros in P, PX and LAST add it to beta
  const Factors* factors;
  bool first;
  // out [rights, lefts] (A, P: [lefts, rights] too, which is the other triangle)
  f16_t* out;
  int64_t out_plane, out_batch;
  int out_planes;
  // LAST: the result [rows, cols] of X's own shape, or its transpose
  void* result;
  int rows, cols;
  bool result_turned;
};

// One workgroup a tile of BL x BR, WL x WR waves, the sums in registers (16 x 16 blocks of v_mfma_f32_16x16x32_f16).
// Slices of 64 of both operands lie in LDS, STAGES of them, filled straight from memory (no registers) STAGES - 1 slices
// ahead.  A wave holds the operands of 32 of a slice's 64 and multiplies them while it reads those of the next 32, so
// LDS and the matrix cores work at once; one barrier a slice.
//
// LDS, an operand by rows: [row][8 pieces of 16 bytes], piece p at p ^ (row % 8): the 8 rows that are read together fall
// on different banks.  X by columns: [k][pieces of 32 bytes = 16 columns], piece p at p ^ key(k), likewise for the 4 + 4
// rows k of a transposing read.  The loads write LDS in lane order, so each lane fetches what belongs at its place.
template <int BL, int BR, int WL, int WR, int STAGES, int PL, int MODE, typename T>
__global__ __launch_bounds__(64 * WL * WR) void ns_product_kernel(Args p) {
  constexpr int THREADS = 64 * WL * WR, BK = 64, TL = BL / WL / 16, TR = BR / WR / 16;
  constexpr bool IS_A = MODE == XXT || MODE == XXT_PART || MODE == XXT_JOIN, SYM = IS_A || MODE == AA;
  constexpr bool COLUMNS = !SYM;  // left by columns
  constexpr int PLANE = (BL + BR) * 128, STAGE = PLANE * PL;
  constexpr int PER = THREADS / 8;         // rows of 128 bytes by one load of the workgroup
  constexpr int PER_K = THREADS * 8 / BL;  // rows k of BL columns by one
  constexpr int LOADS_L = BL / PER, LOADS_P = LOADS_L + BR / PER, LOADS = LOADS_P * PL, READS = PL * (TL + TR);
  static_assert(BL % PER == 0 && BR % PER == 0 && (!COLUMNS || PER_K % 16 == 0) && LOADS * (STAGES - 2) < 64);
  extern __shared__ __align__(1024) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wl = wave / WR, wr = wave % WR;

  // neighbours share operands, on one XCD
  const int tiles = SYM ? p.left_tiles * (p.left_tiles + 1) / 2 : p.left_tiles * p.right_tiles;
  const int all = mfma::xcd_contiguous(blockIdx.x, gridDim.x);
  const int g = MODE == XXT_PART ? __builtin_amdgcn_readfirstlane(all / p.splits) : all;
  const int b = __builtin_amdgcn_readfirstlane(g / tiles), t = g - b * tiles;
  int bl, br;
  if constexpr (SYM) {
    bl = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((bl + 1) * (bl + 2) / 2 <= t) ++bl;
    while (bl * (bl + 1) / 2 > t) --bl;
    br = t - bl * (bl + 1) / 2;
  } else {
    constexpr int G = 4;
    const int group = t / (G * p.left_tiles), rows = min(G, p.right_tiles - group * G), in = t - group * G * p.left_tiles;
    br = group * G + in % rows;
    bl = in / rows;
  }
  bl = __builtin_amdgcn_readfirstlane(bl);
  br = __builtin_amdgcn_readfirstlane(br);

  // where this lane's loads come from: byte offsets from the operands' first slice
  const int64_t ld = (int64_t)p.K * 2, ldx = (int64_t)p.lefts * 2;
  const int piece = ((tid & 7) ^ ((tid >> 3) & 7)) * 16;
  constexpr int PIECES = BL / 8;  // 16-byte pieces of a row k
  // 64 columns: a row is half the banks, so rows of one parity need the keys (with k % 4 a third of the LDS cycles of a
  // float32 P X were conflicts; 4 of 768 x 2048 2 % slower)
  auto key_of = [](int k) { return BL >= 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2); };
  uint32_t from_l[LOADS_L], from_r[BR / PER];
  const char *lp = (const char*)(p.left + b * p.left_batch), *rp = (const char*)(p.right + b * p.right_batch) + br * BR * ld;
  int slices = p.K / BK, split = 0;
  if constexpr (MODE == XXT_PART) {
    split = all - g * p.splits;
    const int first = __builtin_amdgcn_readfirstlane(slices * split / p.splits);
    slices = __builtin_amdgcn_readfirstlane(slices * (split + 1) / p.splits) - first;
    lp += first * (BK * 2);
    rp += first * (BK * 2);
  }
  if constexpr (COLUMNS) {
    const int k = tid / PIECES, at = tid % PIECES, key = key_of(k);
    const int column = bl * BL + ((((at >> 1) ^ key) << 1) | (at & 1)) * 8;
    from_l[0] = (uint32_t)(k * ldx + min(column, p.lefts - 8) * 2);
  } else {
    lp += bl * BL * ld;
#pragma unroll
    for (int i = 0; i < LOADS_L; ++i)
      from_l[i] = (uint32_t)(min(i * PER + (tid >> 3), p.lefts - 1 - bl * BL) * ld + piece);
  }
#pragma unroll
  for (int i = 0; i < BR / PER; ++i)
    from_r[i] = (uint32_t)(min(i * PER + (tid >> 3), p.rights - 1 - br * BR) * ld + piece);
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_char*)lds + wave * 1024;
  auto fetch_one = [&](auto I, int k, int stage) {
    constexpr int pl = I.value / LOADS_P, i = I.value % LOADS_P;
    const uint32_t to = lds_at + stage * STAGE + I.value * (PER * 128);
    if constexpr (i >= LOADS_L)
      to_lds(to, from_r[i - LOADS_L], rp + pl * p.right_plane * 2 + k * (BK * 2));
    else if constexpr (COLUMNS)
      to_lds(to, from_l[0], lp + pl * p.left_plane * 2 + (int64_t)(k * BK + i * PER_K) * ldx);
    else
      to_lds(to, from_l[i], lp + pl * p.left_plane * 2 + k * (BK * 2));
  };

  // A symmetric product of pairs has sums of their own for lo hi and for hi lo: A[l][r] and A[r][l] then have the same
  // bits, and so have the entries of equal rows of X on either side of the diagonal.  (In one running sum they differ by
  // a rounding, which gives equal rows directions of their own: 4e-4 of the norm after ten steps, so 5e-6.)
  constexpr bool APART = SYM && PL == 2 && MODE != XXT_JOIN;
  f32x4 acc[TL][TR], low[2][APART ? TL : 1][APART ? TR : 1];
#pragma unroll
  for (int i = 0; i < TL; ++i)
#pragma unroll
    for (int j = 0; j < TR; ++j) {
      acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (APART) low[0][i][j] = low[1][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

  const int row = lane & 15, quad = lane >> 4;
  struct Half {  // a wave's operands of 32 of a slice's 64
    f16x8 l[PL][TL], r[PL][TR];
  };
  const int by_row = row * 128 + ((quad ^ (row & 7)) << 4);
  const int first_k = quad * 8 + (row >> 2), by_column = first_k * (BL * 2) + (key_of(first_k) ^ (wl * TL)) * 32 + (row & 3) * 8;
  // read I of half s of the slice at LDS offset `base`: 8 values along k, from 32 s + 8 quad, of a row or a column
  auto read_one = [&](auto I, Half& h, int base, int s) {
    constexpr int pl = I.value / (TL + TR), i = I.value % (TL + TR);
    const char* plane = lds + base + pl * PLANE;
    if constexpr (i >= TL) {
      h.r[pl][i - TL] = *(const f16x8*)(plane + BL * 128 + (wr * TR + i - TL) * 2048 + (by_row ^ (s * 64)));
    } else if constexpr (COLUMNS) {
      const char* at = plane + s * (32 * BL * 2) + (by_column ^ (i * 32));
      h.l[pl][i] = __builtin_bit_cast(f16x8, mfma::tr_pair(at, at + 4 * BL * 2));
    } else {
      h.l[pl][i] = *(const f16x8*)(plane + (wl * TL + i) * 2048 + (by_row ^ (s * 64)));
    }
  };
  // one half's products, a row of blocks at a time, each with its share of the next half's reads and of `more`
  auto multiply = [&](const Half& h, Half& next, int next_base, int next_s, auto&& more) {
    mfma::static_for<0, TL>([&](auto I) {
      constexpr int i = I.value;
      mfma::static_for<READS * i / TL, READS * (i + 1) / TL>([&](auto R) { read_one(R, next, next_base, next_s); });
      more(I);
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        if constexpr (PL == 2) {
          f32x4 &lo_hi = APART ? low[0][APART ? i : 0][APART ? j : 0] : acc[i][j],
                &hi_lo = APART ? low[1][APART ? i : 0][APART ? j : 0] : acc[i][j];
          lo_hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(h.l[1][i], h.r[0][j], lo_hi, 0, 0, 0);
          hi_lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(h.l[0][i], h.r[1][j], hi_lo, 0, 0, 0);
        }
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h.l[0][i], h.r[0][j], acc[i][j], 0, 0, 0);
      }
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
  auto part_at = [&](int of, int block) {
    return (f32x4*)p.partial + (((int64_t)g * p.splits + of) * (TL * TR) + block) * THREADS + tid;
  };
  if constexpr (MODE == XXT_JOIN) {
    for (int of = 0; of < p.splits; ++of)
#pragma unroll
      for (int i = 0; i < TL; ++i)
#pragma unroll
        for (int j = 0; j < TR; ++j) acc[i][j] += *part_at(of, i * TR + j);
  } else {
    Half h0, h1;
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k)
      mfma::static_for<0, LOADS>([&](auto I) { fetch_one(I, min(k, slices - 1), k); });
    landed(Behind{});
    mfma::static_for<0, READS>([&](auto R) { read_one(R, h0, 0, 0); });
    mfma::static_for<0, LOADS>([&](auto I) { fetch_one(I, min(STAGES - 1, slices - 1), STAGES - 1); });
    int stage = 0;
    for (int k = 0; k < slices; ++k) {
      const int next = stage + 1 == STAGES ? 0 : stage + 1, ahead = min(k + STAGES, slices - 1);
      multiply(h0, h1, stage * STAGE, 1, [](auto) {});
      landed(Behind{});  // slice k + 1 is there, slice k has been read
      multiply(h1, h0, next * STAGE, 0, [&](auto I) {
        mfma::static_for<LOADS * I.value / TL, LOADS * (I.value + 1) / TL>([&](auto L) { fetch_one(L, ahead, stage); });
      });
      stage = next;
    }
    landed(std::integral_constant<int, 0>{});
    if constexpr (APART) {
#pragma unroll
      for (int i = 0; i < TL; ++i)
#pragma unroll
        for (int j = 0; j < TR; ++j) acc[i][j] += low[0][i][j] + low[1][i][j];
    }
  }
  if constexpr (MODE == XXT_PART) {
#pragma unroll
    for (int i = 0; i < TL; ++i)
#pragma unroll
      for (int j = 0; j < TR; ++j) *part_at(split, i * TR + j) = acc[i][j];
    return;
  }

  // A lane has left 4 quad .. 4 quad + 3 of right `row` of each block.
  const Factors f = p.factors[b];
  const float u = p.first ? f.first : f.later;
  float alpha = p.alpha, beta = p.beta;
  if constexpr (IS_A) alpha *= u * u;
  if constexpr (MODE == PX) {
    alpha *= u / f.later;
    beta *= u / f.later;
  }
  if constexpr (MODE == LAST) {
    alpha *= u;
    beta *= u;
  }
  const int l0 = bl * BL + wl * TL * 16, r0 = br * BR + wr * TR * 16;
  const f16_t* e = p.e + b * p.e_batch;
  float* diagonal = p.diagonal + (int64_t)b * p.rights;
  // 16 rows of [rows, 8 * EACH columns] at a time, turned in the wave's own part of LDS: 16 bytes a lane, whole lines
  constexpr int WIDE = TL > TR ? TL : TR, STRIP = 16 * (WIDE * 16 + 4);
  float* strip = (float*)lds + wave * STRIP;
  auto out_rows = [&](auto BLOCKS, int row0, int rows, int col0, int cols, bool with_e) {
    constexpr int EACH = BLOCKS.value * 2, LDW = BLOCKS.value * 16 + 4;
#pragma unroll
    for (int h = 0; h < (16 * EACH + 63) / 64; ++h) {
      const int at = h * 64 + lane, r = at / EACH, c = at % EACH * 8, m = row0 + r, n = col0 + c;
      if (r >= 16 || m >= rows || n >= cols) continue;
      const f32x4 v0 = *(const f32x4*)(strip + r * LDW + c), v1 = *(const f32x4*)(strip + r * LDW + c + 4);
      float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
      if (with_e) {
        const int64_t from = (int64_t)m * cols + n;
        const f16x8 hi = *(const f16x8*)(e + from);
        f16x8 lo = {};
        if (p.e_planes == 2) lo = *(const f16x8*)(e + p.e_plane + from);
        const float rate = MODE == AA || PL == 2 ? beta : fmaf(alpha, diagonal[m], beta);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = fmaf(rate, (float)hi[q] + (float)lo[q], v[q]);
      }
      if constexpr (MODE == AA && PL == 1)
        if (bl == br) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (m == n + q) {
              diagonal[m] = v[q];
              v[q] = 0.f;
            }
        }
      if constexpr (MODE == LAST) {
        const int R = p.result_turned ? p.cols : p.rows, C = p.result_turned ? p.rows : p.cols;
        if (m >= R || n >= C) continue;
        T* to = (T*)p.result + (int64_t)b * R * C + (int64_t)m * C + n;
        if (n + 8 <= C) {
#pragma unroll
          for (int q = 0; q < 8; q += 16 / sizeof(T)) {
            *(raw_at<T>*)(to + q) = rounded_vec<T>(v + q);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (n + q < C) to[q] = from_f32<T>(v[q]);
        }
      } else {
        store_planes(p.out + b * p.out_batch + (int64_t)m * cols + n, p.out_plane, p.out_planes == 2, v);
      }
    }
  };
  if (!(MODE == LAST && p.result_turned)) {
#pragma unroll
    for (int j = 0; j < TR; ++j) {
      wave_fence();
#pragma unroll
      for (int i = 0; i < TL; ++i) *(f32x4*)(strip + row * (TL * 16 + 4) + i * 16 + quad * 4) = acc[i][j] * alpha;
      wave_fence();
      out_rows(std::integral_constant<int, TL>{}, r0 + j * 16, p.rights, l0, p.lefts, !IS_A);
    }
  }
  if ((SYM && bl != br) || (MODE == LAST && p.result_turned)) {
#pragma unroll
    for (int i = 0; i < TL; ++i) {
      wave_fence();
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        f32x4 v = acc[i][j] * alpha;
        const int l = l0 + i * 16 + quad * 4, r = r0 + j * 16 + row;
        if (MODE == LAST && l < p.lefts && r < p.rights) {  // e lies the other way round
          const int64_t from = (int64_t)r * p.lefts + l;
          const f16x4 hi = *(const f16x4*)(e + from);
          f16x4 lo = {};
          if (p.e_planes == 2) lo = *(const f16x4*)(e + p.e_plane + from);
          const float rate = PL == 2 ? beta : fmaf(alpha, diagonal[r], beta);
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = fmaf(rate, (float)hi[q] + (float)lo[q], v[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) strip[(quad * 4 + q) * (TR * 16 + 4) + j * 16 + row] = v[q];
      }
      wave_fence();
      out_rows(std::integral_constant<int, TR>{}, l0 + i * 16, p.lefts, r0, p.rights, MODE == AA);
    }
  }
}

// ------------------------------------------------------------------------------------------------ small matrices
// A whole matrix in one workgroup and one launch: X [D, N] by rows in LDS (f16 planes), A and then P [D, D] beside it,
// and every wave's part of X in float32 registers.  A lane has left 4 quad .. + 3 of right `row` of a block, which is four
// neighbours of a row of X in P X and, as A and P are symmetric, of theirs: no block is turned.  Pieces of 16 bytes lie
// at piece ^ (row % 8).  Bound by the latency of 3 products and 5 barriers a step: 128 x 128 bf16 in 27 us, where
// the separate launches of the tiled form take 60.
constexpr int SMALL_THREADS = 512, SMALL_WL = 2, SMALL_WR = 4;

template <int D, int N, int PL, bool TALL, typename T>
__global__ __launch_bounds__(SMALL_THREADS) void ns_small_kernel(const T* __restrict__ g, T* __restrict__ out, int rows,
                                                                 int cols, Coefficients co, int steps, double eps,
                                                                 double growth) {
  constexpr int TA = D / SMALL_WL / 16, TX = N / SMALL_WL / 16, TR = D / SMALL_WR / 16;  // blocks of a wave
  constexpr int X_PLANE = D * N * 2, A_PLANE = D * D * 2;
  extern __shared__ __align__(1024) char lds[];
  char *xs = lds, *as = lds + PL * X_PLANE;
  double* sums = (double*)as;
  float* diagonal = (float*)(as + PL * A_PLANE);  // P's
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wl = wave / SMALL_WR, wr = wave % SMALL_WR;
  const int row = lane & 15, quad = lane >> 4;
  g += (int64_t)blockIdx.x * rows * cols;
  out += (int64_t)blockIdx.x * rows * cols;

  // X[m][n .. n + 3] of block (i, j): n = (wl TX + i) 16 + 4 quad, m = (wr TR + j) 16 + row
  float x[TX][TR][4];
  double s = 0.0;
  // Four neighbours by one access where the block is whole (a wide matrix); the loads of all blocks are under way at once.
  // (Value by value they took 16 us of 37 at 128 x 128: 16 lines an access.)
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TR; ++j) {
      const int n = (wl * TX + i) * 16 + 4 * quad, m = (wr * TR + j) * 16 + row, mc = min(m, rows - 1);
      if (!TALL && (wl * TX + i) * 16 + 16 <= cols) {
        const Four<T> v = load_four(g + mc * cols + n);
#pragma unroll
        for (int q = 0; q < 4; ++q) x[i][j][q] = m < rows ? to_f32(v.e[q]) : 0.f;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int nc = min(n + q, cols - 1);
          const float v = to_f32(g[TALL ? nc * rows + mc : mc * cols + nc]);
          x[i][j][q] = m < rows && n + q < cols ? v : 0.f;
        }
      }
    }
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TR; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) s = fma((double)x[i][j][q], (double)x[i][j][q], s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < SMALL_THREADS / 64; ++w) s += sums[w];
  double enter;
  const Factors f = factors_of(sqrt(s), eps, growth, enter);
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TR; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) x[i][j][q] = (float)((double)x[i][j][q] * enter);

  // 8 values along k of a row, from 32 s + 8 quad
  auto by_row = [&](const char* base, int width, int block, int k32) {
    const int r = block * 16 + row;
    return *(const f16x8*)(base + r * (width * 2) + (((k32 * 4 + quad) ^ (r & 7)) << 4));
  };
  // of a column of X
  auto by_column = [&](const char* base, int block, int k32) {
    const int k = k32 * 32 + quad * 8 + (row >> 2), piece = (2 * block + ((row & 3) >> 1)) ^ (row >> 2);
    const char* at = base + k * (N * 2) + (row & 1) * 8;
    return __builtin_bit_cast(f16x8, mfma::tr_pair(at + (piece << 4), at + 4 * (N * 2) + ((piece ^ 4) << 4)));
  };
  auto place = [&](char* base, int width, int r, int c) {  // 4 values at (r, c)
    return base + r * (width * 2) + (((c >> 3) ^ (r & 7)) << 4) + (c & 4) * 2;
  };
  auto put = [&](char* base, int plane, int width, int r, int c, const f32x4& v) {
    f16x4 hi, lo;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      _Float16 h, l;
      split(v[q], h, l);
      hi[q] = h;
      lo[q] = l;
    }
    *(f16x4*)place(base, width, r, c) = hi;
    if constexpr (PL == 2) *(f16x4*)(place(base, width, r, c) + plane) = lo;
  };
  // acc[i][j] = sum over K of the wave's left blocks and its right rows; pairs of a symmetric product as in the tiles
  auto product = [&](auto& acc, auto BLOCKS, auto K, auto SYM, auto&& left, const char* right, int right_plane,
                     int right_width) {
    constexpr bool APART = SYM.value && PL == 2;
    f32x4 low[2][APART ? BLOCKS.value : 1][APART ? TR : 1];
#pragma unroll
    for (int i = 0; i < BLOCKS.value; ++i)
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (APART) low[0][i][j] = low[1][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll 4
    for (int k = 0; k < K.value / 32; ++k) {
      f16x8 r[PL][TR];
#pragma unroll
      for (int pl = 0; pl < PL; ++pl)
#pragma unroll
        for (int j = 0; j < TR; ++j) r[pl][j] = by_row(right + pl * right_plane, right_width, wr * TR + j, k);
#pragma unroll
      for (int i = 0; i < BLOCKS.value; ++i) {
        f16x8 l[PL];
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) l[pl] = left(pl, wl * BLOCKS.value + i, k);
#pragma unroll
        for (int j = 0; j < TR; ++j) {
          if constexpr (PL == 2) {
            f32x4 &lo_hi = APART ? low[0][APART ? i : 0][APART ? j : 0] : acc[i][j],
                  &hi_lo = APART ? low[1][APART ? i : 0][APART ? j : 0] : acc[i][j];
            lo_hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[1], r[0][j], lo_hi, 0, 0, 0);
            hi_lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0], r[1][j], hi_lo, 0, 0, 0);
          }
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0], r[0][j], acc[i][j], 0, 0, 0);
        }
      }
    }
    if constexpr (APART) {
#pragma unroll
      for (int i = 0; i < BLOCKS.value; ++i)
#pragma unroll
        for (int j = 0; j < TR; ++j) acc[i][j] += low[0][i][j] + low[1][i][j];
    }
  };
  using IntA = std::integral_constant<int, TA>;
  using IntX = std::integral_constant<int, TX>;
  using KX = std::integral_constant<int, N>;
  using KA = std::integral_constant<int, D>;
  for (int step = 0; step < steps; ++step) {
    const float u = step ? f.later : f.first;
    __syncthreads();  // X has been read
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int j = 0; j < TR; ++j)
        put(xs, X_PLANE, N, (wr * TR + j) * 16 + row, (wl * TX + i) * 16 + 4 * quad,
            f32x4{x[i][j][0], x[i][j][1], x[i][j][2], x[i][j][3]});
    __syncthreads();
    f32x4 acc[TA][TR];
    product(acc, IntA{}, KX{}, std::true_type{},
            [&](int pl, int block, int k) { return by_row(xs + pl * X_PLANE, N, block, k); }, xs, X_PLANE, N);
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        acc[i][j] *= SCALE_A * u * u;
        put(as, A_PLANE, D, (wr * TR + j) * 16 + row, (wl * TA + i) * 16 + 4 * quad, acc[i][j]);
      }
    __syncthreads();
    f32x4 sq[TA][TR];
    product(sq, IntA{}, KA{}, std::true_type{},
            [&](int pl, int block, int k) { return by_row(as + pl * A_PLANE, D, block, k); }, as, A_PLANE, D);
    __syncthreads();  // A has been read
    const float pb = SCALE_P * co.v[3 * step + 1] / SCALE_A, pc = SCALE_P * co.v[3 * step + 2] / (SCALE_A * SCALE_A);
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        f32x4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          // one plane: A as it was multiplied
          const float a = PL == 1 ? (float)(_Float16)acc[i][j][q] : acc[i][j][q];
          v[q] = fmaf(pb, a, pc * sq[i][j][q]);
          if (PL == 1 && (wr * TR + j) * 16 + row == (wl * TA + i) * 16 + 4 * quad + q) {
            diagonal[(wr * TR + j) * 16 + row] = v[q];
            v[q] = 0.f;
          }
        }
        put(as, A_PLANE, D, (wr * TR + j) * 16 + row, (wl * TA + i) * 16 + 4 * quad, v);
      }
    __syncthreads();
    f32x4 px[TX][TR];
    product(px, IntX{}, KA{}, std::false_type{},
            [&](int pl, int block, int k) { return by_column(xs + pl * X_PLANE, block, k); }, as, A_PLANE, D);
    const bool last = step + 1 == steps, fine = PL == 2 || (step >= 1 && step <= steps - 2);
    const float to = last ? u : u / f.later, a = co.v[3 * step] * to, b = to / SCALE_P;
#pragma unroll
    for (int j = 0; j < TR; ++j) {
      const float rate = PL == 1 ? fmaf(b, diagonal[(wr * TR + j) * 16 + row], a) : a;
#pragma unroll
      for (int i = 0; i < TX; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          x[i][j][q] = fmaf(rate, fine ? x[i][j][q] : (float)(_Float16)x[i][j][q], b * px[i][j][q]);
    }
  }
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TR; ++j) {
      const int n = (wl * TX + i) * 16 + 4 * quad, m = (wr * TR + j) * 16 + row;
      if (m >= rows) continue;
      if (!TALL && n + 4 <= cols) {
        Four<T> v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v.e[q] = from_f32<T>(x[i][j][q]);
        store_four(out + m * cols + n, v);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < cols) out[TALL ? (n + q) * rows + m : m * cols + n + q] = from_f32<T>(x[i][j][q]);
      }
    }
}

// ------------------------------------------------------------------------------------------------ host
constexpr int CUS = 256;
// Parts of X X^T's long sums, where its tiles of 64 x 64 leave CUs idle: a slice of K takes 0.2 us (a pair 0.43) on its
// own, the second launch that adds the parts up 4; a part keeps some slices.  64 x 8000 bf16 153 us whole, 114 so;
// 300 x 5000 152 and 136; 200 x 3000, near the limit, the same.
int splits_of(int64_t batch, int Mp, int Np, int planes) {
  const int64_t t = Mp / 64, tiles = t * (t + 1) / 2 * batch;
  const int slices = Np / 64, least = planes == 1 ? 6 : 4;
  if (slices < (planes == 1 ? 28 : 14) || tiles > CUS / 2) return 1;
  const int64_t most = CUS / tiles;
  return (int)(most < slices / least ? most : slices / least);
}

struct Plan {
  int splits;
  int planes, M, N, Mp, Np;  // M <= N; padded to multiples of 64
  int64_t x, a;              // elements of a plane of X, of A (P), all matrices
  int64_t parts_at, factors_at, x_at[2], a_at, p_at, diagonal_at, partial_at;  // bytes into the workspace
  size_t bytes;
};

int round_up(int v, int to) { return (v + to - 1) / to * to; }

// Whether ns_small_kernel takes matrices of these sizes: what is larger has no room in LDS or registers (128 x 256 of one
// plane spills 34 registers of a lane already).
bool is_small(int M, int N, int planes) {
  return M <= 64 ? N <= 256 : M <= 128 && N <= (planes == 1 ? 256 : 128);
}

Plan plan_of(int64_t batch, int m, int n, int planes) {
  Plan p;
  p.planes = planes;
  p.M = m < n ? m : n;
  p.N = m < n ? n : m;
  if (is_small(p.M, p.N, p.planes)) {  // no workspace
    p.bytes = 0;
    return p;
  }
  p.Mp = round_up(p.M, 64);
  p.Np = round_up(p.N, 64);
  p.x = batch * p.Mp * p.Np;
  p.a = batch * p.Mp * p.Mp;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.parts_at = take(batch * NORM_PARTS * 8);
  p.factors_at = take(batch * (int64_t)sizeof(Factors));
  for (int64_t& x : p.x_at) x = take(2 * p.x * 2);  // X has its lo plane in some steps of one-plane products too
  p.a_at = take(2 * p.a * p.planes);
  p.p_at = take(2 * p.a * p.planes);
  p.diagonal_at = take(p.planes == 1 ? batch * p.Mp * 4 : 0);
  p.splits = splits_of(batch, p.Mp, p.Np, p.planes);
  const int64_t t = p.Mp / 64;
  p.partial_at = take(p.splits > 1 ? batch * (t * (t + 1) / 2) * p.splits * 64 * 64 * 4 : 0);
  p.bytes = (size_t)at;
  return p;
}

template <int BL, int BR, int WL, int WR, int STAGES, int PL, int MODE, typename T>
int launch_tiles(Args a, int64_t batch, hipStream_t st) {
  constexpr int TL = BL / WL / 16, TR = BR / WR / 16;
  constexpr int STRIPS = WL * WR * 16 * ((TL > TR ? TL : TR) * 16 + 4) * 4, SLICES = STAGES * (BL + BR) * 128 * PL;
  constexpr int LDS = SLICES > STRIPS ? SLICES : STRIPS;
  static_assert(LDS <= 160 * 1024);
  auto kernel = ns_product_kernel<BL, BR, WL, WR, STAGES, PL, MODE, T>;
  if (LDS > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "xl_newton_schulz: %s", hipGetErrorString(e));
  }
  a.left_tiles = (a.lefts + BL - 1) / BL;
  a.right_tiles = (a.rights + BR - 1) / BR;
  const bool sym = MODE != PX && MODE != LAST;
  const int64_t tiles = (sym ? (int64_t)a.left_tiles * (a.left_tiles + 1) / 2 : (int64_t)a.left_tiles * a.right_tiles) *
                        (MODE == XXT_PART ? a.splits : 1);
  if (tiles * batch > 0x7fffff) return set_error(XL_ERR_UNSUPPORTED, "xl_newton_schulz: batch too large");
  hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * batch)), dim3(64 * WL * WR), LDS, st, a);
  return check_launch("xl_newton_schulz");
}

// Which tiles.  A tile of 256 x 256 has the best rate of a full chip, smaller ones fill it where there are few tiles, and
// deep stages hide the loads' latency where a CU has one workgroup.  cost: time of a slice of K, in 0.96 us of a 4096^3
// product, from the tiles a CU gets (r); measured (us):
//   bf16, X of 4096 x 4096, P X:   256: 110;  128, 2 stages: 133, 4 stages: 159;  64, 2 stages: 205, 4 stages: 204
//   X X^T there:                   192 (253 tiles): 67;  256 (136): 76;  128 (528): 96;  64 (2080): 128
//   12 of 1024 x 2048, P X:        128 (1536): 69;  256 (384): 72;  64: 90;   X X^T: 128 (432): 33;  192 (252): 36
//   2048 x 5504, P X:              256 (176): 52;  128 (688): 60;  64 (2752): 73
//   X X^T there:                   128, 4 stages (136): 41, 2 stages: 55;  64, 2 stages (528): 47, 4 stages: 62
//   1024 x 1024, P X:              64, 4 stages (256): 8.1, 2 stages: 10.9;  128, 4 stages (64): 14.6
//   float32, 2048 x 2048, P X:     128 (256): 48;  64, 2 stages (1024): 59, 4 stages: 64
//   float32, 1000 x 1777, P X:     64, 2 stages (448): 16.7, 4 stages: 19.3;  128 (112): 26
//   X X^T and A A there:           64, 4 stages (136): 25, 2 stages: 35;  128 (36): 53
//   2048 x 2048, all five steps, X X^T and A A by 128 (136): 643;  64, 2 stages (528): 758, 4 stages: 791
template <int PL, int MODE, typename T>
int launch_product(const Args& a, int64_t batch, hipStream_t st) {
  constexpr bool SYM = MODE == XXT || MODE == AA;
  if constexpr (MODE == XXT)
    if (a.splits > 1) {
      const int rc = launch_tiles<64, 64, 2, 2, 4, PL, XXT_PART, T>(a, batch, st);
      return rc ? rc : launch_tiles<64, 64, 2, 2, 4, PL, XXT_JOIN, T>(a, batch, st);
    }
  auto tiles = [&](int tile) {
    const int64_t l = (a.lefts + tile - 1) / tile, r = (a.rights + tile - 1) / tile;
    return (SYM ? l * (l + 1) / 2 : l * r) * batch;
  };
  auto rounds = [&](int tile) { return (double)((tiles(tile) + CUS - 1) / CUS); };
  auto at_least = [](double v, double least) { return v > least ? v : least; };
  enum { T256, T192, T128_2, T128_4, T64_2, T64_4, CHOICES };
  double cost[CHOICES];
  for (double& c : cost) c = INFINITY;
  if (PL == 1) {
    const double r = rounds(256);
    cost[T256] = 52.4 * r * (0.75 + 0.25 * (double)tiles(256) / (CUS * r));  // a chip not full runs faster
    if (SYM) cost[T192] = 33.5 * rounds(192);
    cost[T128_2] = at_least(16.2 * rounds(128), 19.3);
    cost[T128_4] = (rounds(128) > 1 ? 19.0 : 14.6) * rounds(128);
    cost[T64_2] = at_least(6.1 * rounds(64), 12.8);
    cost[T64_4] = (rounds(64) > 1 ? 7.0 : 8.0) * rounds(64);
  } else {
    cost[T128_2] = 16.4 * rounds(128);
    cost[T64_2] = at_least(5.6 * rounds(64), 9.1);
    cost[T64_4] = 6.2 * rounds(64);
  }
  int best = T128_2;
  for (int c = 0; c < CHOICES; ++c)
    if (cost[c] < cost[best]) best = c;
  if constexpr (PL == 1) {
    if (best == T256) return launch_tiles<256, 256, 2, 4, 2, PL, MODE, T>(a, batch, st);
    if constexpr (SYM)
      if (best == T192) return launch_tiles<192, 192, 2, 4, 2, PL, MODE, T>(a, batch, st);
    if (best == T128_4) return launch_tiles<128, 128, 2, 2, 4, PL, MODE, T>(a, batch, st);
  }
  if (best == T64_2) return launch_tiles<64, 64, 2, 2, 2, PL, MODE, T>(a, batch, st);
  // A symmetric product of pairs has three sums a block: 8 waves, each of half as many blocks.  us for all steps, float32:
  // 2048 x 2048 662, with 4 waves 819 (more than 256 registers, which the compiler moves about); 1777 x 1000 228 and 235.
  // Tiles of 64 with two stages, two workgroups a CU, stay with 4: 4 of 768 x 2048 440, with 8 443.
  if constexpr (SYM && PL == 2) {
    if (best == T64_4) return launch_tiles<64, 64, 2, 4, 4, PL, MODE, T>(a, batch, st);
    return launch_tiles<128, 128, 2, 4, 2, PL, MODE, T>(a, batch, st);
  }
  if (best == T64_4) return launch_tiles<64, 64, 2, 2, 4, PL, MODE, T>(a, batch, st);
  return launch_tiles<128, 128, 2, 2, 2, PL, MODE, T>(a, batch, st);
}

template <int D, int N, int PL, typename T>
int launch_small(const void* g, void* x, int64_t batch, int m, int n, const Coefficients& co, int steps, float eps,
                 double growth, hipStream_t st) {
  constexpr int LDS = PL * (D * N + D * D) * 2 + D * 4;
  static_assert(LDS <= 160 * 1024);
  auto kernel = m > n ? ns_small_kernel<D, N, PL, true, T> : ns_small_kernel<D, N, PL, false, T>;
  if (LDS > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "xl_newton_schulz: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)batch), dim3(SMALL_THREADS), LDS, st, (const T*)g, (T*)x, m < n ? m : n,
                     m < n ? n : m, co, steps, (double)eps, growth);
  return check_launch("xl_newton_schulz");
}

template <typename T, int PL>
int run_small(const void* g, void* x, int64_t batch, int m, int n, const Coefficients& co, int steps, float eps, double growth,
              hipStream_t st) {
  const int M = m < n ? m : n, N = m < n ? n : m;
  if (M <= 64) {
    if (N <= 64) return launch_small<64, 64, PL, T>(g, x, batch, m, n, co, steps, eps, growth, st);
    if (N <= 128) return launch_small<64, 128, PL, T>(g, x, batch, m, n, co, steps, eps, growth, st);
    return launch_small<64, 256, PL, T>(g, x, batch, m, n, co, steps, eps, growth, st);
  }
  if constexpr (PL == 1) {
    if (N > 128) return launch_small<128, 256, PL, T>(g, x, batch, m, n, co, steps, eps, growth, st);
  }
  return launch_small<128, 128, PL, T>(g, x, batch, m, n, co, steps, eps, growth, st);
}

template <typename T, int PL>
int run(const void* g, void* x, int64_t batch, int m, int n, const float* coefficients, int steps, float eps, double growth,
        const Plan& p, char* ws, hipStream_t st) {
  if (is_small(p.M, p.N, PL)) {
    Coefficients co;
    for (int i = 0; i < 3 * steps; ++i) co.v[i] = coefficients[i];
    return run_small<T, PL>(g, x, batch, m, n, co, steps, eps, growth, st);
  }
  const bool tall = m > n;
  double* part = (double*)(ws + p.parts_at);
  Factors* factors = (Factors*)(ws + p.factors_at);
  f16_t *X[2] = {(f16_t*)(ws + p.x_at[0]), (f16_t*)(ws + p.x_at[1])}, *A = (f16_t*)(ws + p.a_at), *P = (f16_t*)(ws + p.p_at);
  const int64_t count = (int64_t)m * n;
  const int64_t want = (count + 64 * NORM_BLOCK - 1) / (64 * NORM_BLOCK);
  const int parts = (int)(want < NORM_PARTS ? want : NORM_PARTS);
  hipLaunchKernelGGL(ns_norm_kernel<T>, dim3((unsigned)parts, (unsigned)batch), dim3(NORM_BLOCK), 0, st, (const T*)g, count,
                     parts, part);
  auto enter = tall ? ns_enter_kernel<T, PL, true> : ns_enter_kernel<T, PL, false>;
  hipLaunchKernelGGL(enter, dim3((unsigned)(p.Np / 64), (unsigned)(p.Mp / 64), (unsigned)batch), dim3(256), 0, st, (const T*)g,
                     p.M, p.N, p.Mp, p.Np, part, parts, (double)eps, growth, X[0], p.x, factors);
  if (const int rc = check_launch("xl_newton_schulz")) return rc;
  const int64_t xb = (int64_t)p.Mp * p.Np, ab = (int64_t)p.Mp * p.Mp;
  for (int s = 0; s < steps; ++s) {
    const float a = coefficients[3 * s], b = coefficients[3 * s + 1], c = coefficients[3 * s + 2];
    const bool last = s + 1 == steps;
    // a X in more bits than the products': what rounding leaves in the directions of small singular values grows 3.4-fold
    // a step with them.  In every step but the first, which is exact, and the last, after which nothing grows.  (Matrices
    // of rank 8, rounded to bf16, 128 x 256: 2.5e-3 so, 3.3e-3 without the step before the last, 6.6e-3 in step 1 alone.)
    auto fine = [&](int step) { return PL == 2 || (step >= 1 && step <= steps - 2); };
    const f16_t* old = X[s & 1];
    Args k{};
    k.factors = factors;
    k.first = s == 0;
    k.diagonal = (float*)(ws + p.diagonal_at);
    k.left = k.right = old;
    k.left_plane = k.right_plane = p.x;
    k.left_batch = k.right_batch = xb;
    k.lefts = k.rights = p.Mp;
    k.K = p.Np;
    k.splits = p.splits;
    k.partial = (float*)(ws + p.partial_at);
    k.alpha = SCALE_A;
    k.out = A;
    k.out_plane = p.a;
    k.out_batch = ab;
    k.out_planes = PL;
    if (const int rc = launch_product<PL, XXT, T>(k, batch, st)) return rc;
    k.left = k.right = k.e = A;
    k.left_plane = k.right_plane = k.e_plane = p.a;
    k.left_batch = k.right_batch = k.e_batch = ab;
    k.e_planes = PL;
    k.K = p.Mp;
    k.alpha = SCALE_P * c / (SCALE_A * SCALE_A);
    k.beta = SCALE_P * b / SCALE_A;
    k.out = P;
    if (const int rc = launch_product<PL, AA, T>(k, batch, st)) return rc;
    k.left = k.e = old;
    k.left_plane = k.e_plane = p.x;
    k.left_batch = k.e_batch = xb;
    k.e_planes = fine(s) ? 2 : 1;
    k.right = P;
    k.lefts = p.Np;
    k.alpha = 1.f / SCALE_P;
    k.beta = a;
    k.out = X[(s + 1) & 1];
    k.out_plane = p.x;
    k.out_batch = xb;
    k.out_planes = fine(s + 1) ? 2 : 1;
    k.result = x;
    k.rows = p.M;
    k.cols = p.N;
    k.result_turned = tall;
    if (const int rc = last ? launch_product<PL, LAST, T>(k, batch, st) : launch_product<PL, PX, T>(k, batch, st)) return rc;
  }
  return XL_OK;
}

int check_sizes(const char* who, int64_t batch, int m, int n, int dtype) {
  if (batch < 0 || m < 0 || n < 0)
    return set_error(XL_ERR_INVALID_ARG, "%s: negative size (batch=%lld m=%d n=%d)", who, (long long)batch, m, n);
  if (!dtype_ok(dtype)) return set_error(XL_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
  if (m > 65536 || n > 65536 || batch > 65535)
    return set_error(XL_ERR_UNSUPPORTED, "%s: batch=%lld m=%d n=%d (at most 65535 matrices of 65536 x 65536)", who,
                     (long long)batch, m, n);
  return XL_OK;
}

// what any coefficients take: bf16 runs one plane or pairs
size_t workspace_of(int64_t batch, int m, int n, int dtype) {
  const size_t pairs = plan_of(batch, m, n, 2).bytes, one = dtype == XL_DTYPE_BF16 ? plan_of(batch, m, n, 1).bytes : 0;
  return one > pairs ? one : pairs;
}

}  // namespace
}  // namespace xl

extern "C" size_t xl_newton_schulz_workspace_size(int64_t batch, int m, int n, int dtype) {
  using namespace xl;
  if (check_sizes("xl_newton_schulz_workspace_size", batch, m, n, dtype) || batch == 0 || m == 0 || n == 0) return 0;
  return workspace_of(batch, m, n, dtype);
}

extern "C" int xl_newton_schulz(const void* g, void* x, int64_t batch, int m, int n, const float* coefficients, int steps,
                                float eps, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace xl;
  clear_error();
  const char* who = "xl_newton_schulz";
  if (const int rc = check_sizes(who, batch, m, n, dtype)) return rc;
  if (steps < 1 || steps > MOST_STEPS || !coefficients)
    return set_error(XL_ERR_INVALID_ARG, "%s: steps=%d (1 to %d, with coefficients)", who, steps, MOST_STEPS);
  if (!(eps >= 0.f)) return set_error(XL_ERR_INVALID_ARG, "%s: eps=%g (not negative)", who, (double)eps);
  // singular values start in [0, 1]: the most that a step's polynomial makes of them, and of what was rounded before it; and
  // by how much a small one can have grown
  double most = 1.0, noise = 0.0, growth = 1.0;
  for (int s = 0; s < steps; ++s) {
    const double a = coefficients[3 * s], b = coefficients[3 * s + 1], c = coefficients[3 * s + 2], x2 = most * most;
    const double in_p = fabs(b) * x2 + fabs(c) * x2 * x2;
    double next = 0.0, slope = 1.0, rate = 1.0;
    for (int i = 0; i <= 1024; ++i) {
      const double v = most * i / 1024, v2 = v * v, by = fabs(a + b * v2 + c * v2 * v2), y = v * by;
      if (!(y <= next)) next = y;
      rate = fmax(rate, by);
      slope = fmax(slope, fabs(a + 3.0 * b * v2 + 5.0 * c * v2 * v2));
    }
    noise = noise * slope + 1.0;
    growth *= rate;
    if (!(in_p <= MOST_P) || !(next <= 0.99 * MOST_X))
      return set_error(XL_ERR_INVALID_ARG, "%s: step %d's coefficients (%g, %g, %g) take singular values out of range", who, s, a,
                       b, c);
    most = next * 1.01;  // between the samples, and the products' rounding
  }
  if (batch == 0 || m == 0 || n == 0) return XL_OK;
  if (!g || !x) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (g == x) return set_error(XL_ERR_INVALID_ARG, "%s: x must not alias g", who);
  const size_t need = workspace_of(batch, m, n, dtype);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255u)))
    return set_error(XL_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", who, need,
                     workspace_bytes);
  const Plan p = plan_of(batch, m, n, dtype == XL_DTYPE_BF16 && noise <= MOST_NOISE ? 1 : 2);
  char* ws = (char*)workspace;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case XL_DTYPE_F32: return run<float, 2>(g, x, batch, m, n, coefficients, steps, eps, growth, p, ws, st);
    case XL_DTYPE_BF16:
      return p.planes == 1 ? run<bf16_t, 1>(g, x, batch, m, n, coefficients, steps, eps, growth, p, ws, st)
                           : run<bf16_t, 2>(g, x, batch, m, n, coefficients, steps, eps, growth, p, ws, st);
    default: return run<f16_t, 2>(g, x, batch, m, n, coefficients, steps, eps, growth, p, ws, st);
  }
}
