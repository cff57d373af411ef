// Orthogonalisation of a matrix by Newton-Schulz products:
//
//   X = G / (|G|_F + eps);  steps times:  A = X X^T,  P = b A + c A^2,  X = a X + P X
//
// on the side with fewer rows (G^T for a tall G), so that every singular value s goes to s (a + b s^2 + c s^4) a step.
// The products are on the matrix cores in f16 with float32 sums.  Every matrix is kept at a power-of-two scale that
// holds it in f16's range; a bf16 G enters exactly, its results' own rounding (1.65e-3 of the norm) is larger than what
// the f16 intermediates add (bf16 intermediates: 1e-2 to 3e-2).  For f16 and float32 every matrix is a pair
// hi + lo of f16 (22 bits) and a product three (hi hi + hi lo + lo hi), 4e-7 of the norm.
//
// A and P are symmetric: their tiles on and below the diagonal are computed and written to both places.  X is kept
// as X and X^T, so that all three products have both operands' sums along contiguous rows (X X^T, A A, P (X^T)^T).
// All matrices are zero-padded to whole tiles in the workspace: no bounds in the loops, and products of zeros stay
// zero.
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
typedef __attribute__((address_space(3))) char lds_char;

// stored = value * scale: with |singular values| of X up to 8 (checked on the host), |A| <= 64 and |P| <= 250
constexpr float SCALE_X = 256.f, SCALE_A = 256.f, SCALE_P = 64.f;
constexpr float MOST_X = 8.f, MOST_P = 250.f;

// ------------------------------------------------------------------------------------------------ norm and first X
constexpr int NORM_BLOCK = 256, NORM_PARTS = 256;  // partial sums per matrix

template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void ns_norm_kernel(const T* __restrict__ g, int64_t count, int parts,
                                                             double* __restrict__ part) {
  __shared__ double sums[NORM_BLOCK / 64];
  const T* p = g + blockIdx.y * count;
  double s = 0.0;  // no float32 value's square overflows it
  for (int64_t i = (int64_t)blockIdx.x * NORM_BLOCK + threadIdx.x; i < count; i += (int64_t)parts * NORM_BLOCK) {
    const double v = (double)to_f32(p[i]);
    s = fma(v, v, s);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)blockIdx.y * parts + blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

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
  // a G far below eps keeps its smallness: it is scaled up by what the steps cannot make up for
  int up = 0;
  const double share = norm / (norm + eps) * growth;
  if (share > 0.0 && share < 1.0) {
    frexp(share, &up);
    up = up < -100 ? 100 : up < 0 ? -up : 0;
  }
  return Factors{(float)(1.0 / ((norm + eps) * enter)), (float)ldexp(1.0 / SCALE_X, -up)};
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// G [R, C] into `same` [Rp, Cp] and `turned` [Cp, Rp] (f16 planes, zero past G), 64 x 64 a workgroup
template <typename T, int PL>
__global__ __launch_bounds__(256) void ns_enter_kernel(const T* __restrict__ g, int R, int C, int Rp, int Cp,
                                                       const double* __restrict__ part, int parts, double eps,
                                                       double growth, f16_t* __restrict__ same, int64_t same_plane,
                                                       f16_t* __restrict__ turned, int64_t turned_plane,
                                                       Factors* __restrict__ factors) {
  __shared__ float tile[64][65];
  __shared__ double sums[4];
  const int tid = threadIdx.x, b = blockIdx.z;
  double s = tid < parts ? part[(int64_t)b * parts + tid] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((tid & 63) == 0) sums[tid >> 6] = s;
  __syncthreads();
  double enter;
  const Factors f = factors_of(sqrt(sums[0] + sums[1] + sums[2] + sums[3]), eps, growth, enter);
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) factors[b] = f;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, x = tid & 63, y = tid >> 6;
  const T* gp = g + (int64_t)b * R * C;
  const int64_t at = (int64_t)b * Rp * Cp;
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    const int r = r0 + i + y, c = c0 + x;
    const float v = r < R && c < C ? (float)((double)to_f32(gp[(int64_t)r * C + c]) * enter) : 0.f;
    tile[i + y][x] = v;
    _Float16 hi, lo;
    split(v, hi, lo);
    same[at + (int64_t)r * Cp + c] = hi;
    if constexpr (PL == 2) same[same_plane + at + (int64_t)r * Cp + c] = lo;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    _Float16 hi, lo;
    split(tile[x][i + y], hi, lo);
    const int64_t to = at + (int64_t)(c0 + i + y) * Rp + r0 + x;
    turned[to] = hi;
    if constexpr (PL == 2) turned[turned_plane + to] = lo;
  }
}

// ------------------------------------------------------------------------------------------------ the products
// 16 bytes a lane from global memory into LDS, at lds + 16 * lane (lds the same in the whole wave)
__device__ __forceinline__ void to_lds(uint32_t lds, uint32_t offset, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

enum Product { XXT, AA, PX, LAST };  // A; P; X and X^T; the result

struct Args {
  // left [tm BM, K] and right [tn BN, K], planes hi and (plane elements on) lo
  const f16_t *left, *right;
  int64_t left_plane, right_plane, left_batch, right_batch;
  int K, tm, tn;
  // value = beta * e + alpha * sum; e transposed, [tn BN, tm BM], of e_planes
  const f16_t* e;
  int64_t e_plane, e_batch;
  int e_planes;
  float alpha, beta;
  const Factors* factors;
  bool first;
  // out [tm BM, tn BN] and turned [tn BN, tm BM], with out_planes and turned_planes
  f16_t *out, *turned;
  int64_t out_plane, turned_plane, out_batch, turned_batch;
  int out_planes, turned_planes;
  // LAST: the result, [rows, cols], or [cols, rows] where it is turned
  void* result;
  int rows, cols;
  bool result_turned;
};

// One workgroup a tile of BM x BN, WM x WN waves, the sums in registers (16 x 16 blocks of v_mfma_f32_16x16x32_f16).
// Slices of 64 of both operands are in LDS twice: the next one is on its way (straight from memory, no registers)
// while this one is multiplied; one barrier a slice.  A row's 8 pieces of 16 bytes lie at piece ^ (row % 8), so that the
// rows that the matrix cores' lanes read together fall on different banks; as the loads write LDS in lane order,
// each lane fetches the piece that belongs at its place.
template <int BM, int BN, int WM, int WN, int PL, int MODE, typename T>
__global__ __launch_bounds__(64 * WM * WN) void ns_product_kernel(Args p) {
  constexpr int THREADS = 64 * WM * WN, BK = 64, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * BK * 2 * PL, PER = THREADS / 8;  // rows by one load of the workgroup
  constexpr int STRIP = 16 * (TN * 16 + 4) * 4;
  constexpr int LDS = 2 * STAGE > WM * WN * STRIP ? 2 * STAGE : WM * WN * STRIP;
  static_assert(BM % PER == 0 && BN % PER == 0);
  extern __shared__ __align__(1024) char lds[];
  static_assert(LDS <= 160 * 1024);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  constexpr bool SYM = MODE == XXT || MODE == AA;

  // neighbours share rows and columns of tiles, on one XCD
  const int t = mfma::xcd_contiguous(blockIdx.x, gridDim.x), b = blockIdx.y;
  int bi, bj;
  if constexpr (SYM) {
    bi = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
    while (bi * (bi + 1) / 2 > t) --bi;
    bj = t - bi * (bi + 1) / 2;
  } else {
    constexpr int G = 4;
    const int group = t / (G * p.tn), rows = min(G, p.tm - group * G), in = t - group * G * p.tn;
    bi = group * G + in % rows;
    bj = in / rows;
  }
  bi = __builtin_amdgcn_readfirstlane(bi);
  bj = __builtin_amdgcn_readfirstlane(bj);

  const int64_t ld = (int64_t)p.K * 2;
  const uint32_t offset = (uint32_t)((tid >> 3) * ld) + (uint32_t)(((tid & 7) ^ ((tid >> 3) & 7)) * 16);
  const char *lp = (const char*)(p.left + b * p.left_batch) + bi * BM * ld,
             *rp = (const char*)(p.right + b * p.right_batch) + bj * BN * ld;
  const uint32_t at = (uint32_t)(uintptr_t)(lds_char*)lds + wave * 1024;
  auto fetch = [&](int k, int stage) {
    uint32_t to = at + stage * STAGE;
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) {
#pragma unroll
      for (int i = 0; i < BM / PER; ++i, to += PER * 128)
        to_lds(to, offset, lp + pl * p.left_plane * 2 + i * PER * ld + k * (BK * 2));
#pragma unroll
      for (int i = 0; i < BN / PER; ++i, to += PER * 128)
        to_lds(to, offset, rp + pl * p.right_plane * 2 + i * PER * ld + k * (BK * 2));
    }
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int row = lane & 15, quad = lane >> 4;
  auto operand = [&](int base, int r, int s) {  // 8 values of row r, from 32 s + 8 quad
    return *(const f16x8*)(lds + base + r * 128 + (((s * 4 + quad) ^ (r & 7)) << 4));
  };
  const int slices = p.K / BK;
  fetch(0, 0);
  for (int k = 0; k < slices; ++k) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // slice k is there, slice k - 1 has been read
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (k + 1 < slices) fetch(k + 1, (k + 1) & 1);
    const int base = (k & 1) * STAGE;
#pragma unroll
    for (int s = 0; s < BK / 32; ++s) {
      f16x8 l[PL][TM], r[PL][TN];
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) {
        const int at_plane = base + pl * (BM + BN) * 128;
#pragma unroll
        for (int i = 0; i < TM; ++i) l[pl][i] = operand(at_plane, (wm * TM + i) * 16 + row, s);
#pragma unroll
        for (int j = 0; j < TN; ++j) r[pl][j] = operand(at_plane + BM * 128, (wn * TN + j) * 16 + row, s);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if constexpr (PL == 2) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[1][i], r[0][j], acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0][i], r[1][j], acc[i][j], 0, 0, 0);
          }
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0][i], r[0][j], acc[i][j], 0, 0, 0);
        }
    }
  }

  // A lane has rows 4 quad .. 4 quad + 3 of column `row` of each block: four neighbours of a row of the transposed.
  const Factors f = p.factors[b];
  const float u = p.first ? f.first : f.later;
  float alpha = p.alpha, beta = p.beta;
  if constexpr (MODE == XXT) alpha *= u * u;
  if constexpr (MODE == PX) {
    alpha *= u / f.later;
    beta *= u / f.later;
  }
  if constexpr (MODE == LAST) {
    alpha *= u;
    beta *= u;
  }
  const int m0 = bi * BM + wm * TM * 16, n0 = bj * BN + wn * TN * 16;
  const int64_t ldt = (int64_t)p.tm * BM, ldo = (int64_t)p.tn * BN;
  if constexpr (MODE != XXT) {
    const f16_t* e = p.e + b * p.e_batch;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t from = (n0 + j * 16 + row) * ldt + m0 + i * 16 + quad * 4;
        const f16x4 hi = *(const f16x4*)(e + from);
        f16x4 lo = {};
        if (p.e_planes == 2) lo = *(const f16x4*)(e + p.e_plane + from);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][j][q] = fmaf(beta, (float)hi[q] + (float)lo[q], alpha * acc[i][j][q]);
      }
  } else {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] *= alpha;
  }

  const bool by_columns = MODE == LAST ? p.result_turned : true, by_rows = MODE == LAST ? !p.result_turned : true;
  if (by_columns && !(SYM && bi == bj)) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + j * 16 + row, m = m0 + i * 16 + quad * 4;
        if constexpr (MODE == LAST) {
          T* to = (T*)p.result + (int64_t)b * p.rows * p.cols + (int64_t)n * p.rows + m;
          if (n < p.cols) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (m + q < p.rows) to[q] = from_f32<T>(acc[i][j][q]);
          }
        } else {
          f16_t* to = p.turned + b * p.turned_batch + n * ldt + m;
          f16x4 hi, lo;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            _Float16 h, l;
            split(acc[i][j][q], h, l);
            hi[q] = h;
            lo[q] = l;
          }
          *(f16x4*)to = hi;
          if (p.turned_planes == 2) *(f16x4*)(to + p.turned_plane) = lo;
        }
      }
  }
  if (by_rows) {  // 16 rows at a time turned in the wave's own part of LDS
    __syncthreads();
    float* strip = (float*)(lds + wave * STRIP);
    constexpr int LDW = TN * 16 + 4, EACH = TN * 16 / 8;  // 8 values a lane: EACH lanes a row
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      wave_fence();
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) strip[(quad * 4 + q) * LDW + j * 16 + row] = acc[i][j][q];
      wave_fence();
#pragma unroll
      for (int h = 0; h < 16 * EACH / 64; ++h) {
        const int r = h * (64 / EACH) + lane / EACH, c = lane % EACH * 8;
        const f32x4 v0 = *(const f32x4*)(strip + r * LDW + c), v1 = *(const f32x4*)(strip + r * LDW + c + 4);
        const int m = m0 + i * 16 + r, n = n0 + c;
        if constexpr (MODE == LAST) {
          if (m < p.rows) {
            T* to = (T*)p.result + (int64_t)b * p.rows * p.cols + (int64_t)m * p.cols + n;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (n + q < p.cols) to[q] = from_f32<T>(q < 4 ? v0[q] : v1[q - 4]);
          }
        } else {
          f16_t* to = p.out + b * p.out_batch + m * ldo + n;
          f16x8 hi, lo;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            _Float16 a, l;
            split(q < 4 ? v0[q] : v1[q - 4], a, l);
            hi[q] = a;
            lo[q] = l;
          }
          *(f16x8*)to = hi;
          if (p.out_planes == 2) *(f16x8*)(to + p.out_plane) = lo;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
struct Plan {
  int planes, tile, M, N, Mp, Np;  // M <= N; padded to whole tiles
  int64_t x, xt, a;                // elements of a plane of X (X^T), of A (P), all matrices
  int64_t parts_at, factors_at, x_at, xt_at[2], a_at, p_at;  // bytes into the workspace
  size_t bytes;
};

int round_up(int v, int to) { return (v + to - 1) / to * to; }

Plan plan_of(int64_t batch, int m, int n, int dtype) {
  Plan p;
  p.planes = dtype == XL_DTYPE_BF16 ? 1 : 2;
  p.M = m < n ? m : n;
  p.N = m < n ? n : m;
  p.tile = 128;
  p.Mp = round_up(p.M, p.tile);
  p.Np = round_up(p.N, p.tile);
  p.x = batch * p.Mp * p.Np;
  p.xt = p.x;
  p.a = batch * p.Mp * p.Mp;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.parts_at = take(batch * NORM_PARTS * 8);
  p.factors_at = take(batch * (int64_t)sizeof(Factors));
  p.x_at = take(2 * p.x * p.planes);
  for (int64_t& t : p.xt_at) t = take(2 * p.xt * 2);  // X^T has its lo plane in some steps of one-plane products too
  p.a_at = take(2 * p.a * p.planes);
  p.p_at = take(2 * p.a * p.planes);
  p.bytes = (size_t)at;
  return p;
}

template <int BM, int BN, int WM, int WN, int PL, int MODE, typename T>
int launch_product(const Args& a, int64_t batch, hipStream_t st) {
  constexpr int STAGE = (BM + BN) * 128 * PL, STRIP = 16 * (BN / WN + 4) * 4;
  constexpr int LDS = 2 * STAGE > WM * WN * STRIP ? 2 * STAGE : WM * WN * STRIP;
  auto kernel = ns_product_kernel<BM, BN, WM, WN, PL, MODE, T>;
  if (LDS > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return set_error(XL_ERR_LAUNCH, "xl_newton_schulz: %s", hipGetErrorString(e));
  }
  const int tiles = MODE == XXT || MODE == AA ? a.tm * (a.tm + 1) / 2 : a.tm * a.tn;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)batch), dim3(64 * WM * WN), LDS, st, a);
  return check_launch("xl_newton_schulz");
}

template <typename T, int PL>
int run(const void* g, void* x, int64_t batch, int m, int n, const float* coefficients, int steps, float eps, const Plan& p,
        char* ws, hipStream_t st) {
  const bool tall = m > n;
  double* part = (double*)(ws + p.parts_at);
  Factors* factors = (Factors*)(ws + p.factors_at);
  f16_t *X = (f16_t*)(ws + p.x_at), *XT[2] = {(f16_t*)(ws + p.xt_at[0]), (f16_t*)(ws + p.xt_at[1])};
  f16_t *A = (f16_t*)(ws + p.a_at), *P = (f16_t*)(ws + p.p_at);
  const int64_t count = (int64_t)m * n;
  const int64_t want = (count + 16 * NORM_BLOCK - 1) / (16 * NORM_BLOCK);
  const int parts = (int)(want < NORM_PARTS ? want : NORM_PARTS);
  double growth = 1.0;
  for (int s = 0; s < steps; ++s) {
    const double a = fabs((double)coefficients[3 * s]);
    if (a > 1.0) growth *= a;
  }
  hipLaunchKernelGGL(ns_norm_kernel<T>, dim3((unsigned)parts, (unsigned)batch), dim3(NORM_BLOCK), 0, st, (const T*)g, count,
                     parts, part);
  const int Rp = tall ? p.Np : p.Mp, Cp = tall ? p.Mp : p.Np;
  f16_t *same = tall ? XT[0] : X, *turned = tall ? X : XT[0];
  const int64_t x_plane = p.x, xt_plane = p.xt;
  hipLaunchKernelGGL((ns_enter_kernel<T, PL>), dim3((unsigned)(Cp / 64), (unsigned)(Rp / 64), (unsigned)batch), dim3(256), 0, st,
                     (const T*)g, m, n, Rp, Cp, part, parts, (double)eps, growth, same, tall ? xt_plane : x_plane, turned,
                     tall ? x_plane : xt_plane, factors);
  if (const int rc = check_launch("xl_newton_schulz")) return rc;
  const int64_t xb = (int64_t)p.Mp * p.Np, ab = (int64_t)p.Mp * p.Mp;
  for (int s = 0; s < steps; ++s) {
    const float a = coefficients[3 * s], b = coefficients[3 * s + 1], c = coefficients[3 * s + 2];
    const bool last = s + 1 == steps;
    // a X in more bits than the products' while the smallest singular values grow: to the step before the last two.
    // Later the rounding of X is better the same in both terms: there the steps contract, and correct it.
    auto fine = [&](int step) { return PL == 2 || (step >= 1 && step <= steps - 3); };
    const f16_t* old = XT[s & 1];
    f16_t* next = XT[(s + 1) & 1];
    Args k{};
    k.factors = factors;
    k.first = s == 0;
    k.left = k.right = X;
    k.left_plane = k.right_plane = p.x;
    k.left_batch = k.right_batch = xb;
    k.K = p.Np;
    k.tm = k.tn = p.Mp / p.tile;
    k.alpha = SCALE_A;
    k.out = k.turned = A;
    k.out_plane = k.turned_plane = p.a;
    k.out_batch = k.turned_batch = ab;
    k.out_planes = k.turned_planes = PL;
    if (const int rc = launch_product<128, 128, 2, 2, PL, XXT, T>(k, batch, st)) return rc;
    k.left = k.right = k.e = A;
    k.left_plane = k.right_plane = k.e_plane = p.a;
    k.left_batch = k.right_batch = k.e_batch = ab;
    k.e_planes = PL;
    k.K = p.Mp;
    k.alpha = SCALE_P * c / (SCALE_A * SCALE_A);
    k.beta = SCALE_P * b / SCALE_A;
    k.out = k.turned = P;
    if (const int rc = launch_product<128, 128, 2, 2, PL, AA, T>(k, batch, st)) return rc;
    k.left = P;
    k.right = k.e = old;
    k.right_plane = k.e_plane = p.xt;
    k.right_batch = k.e_batch = xb;
    k.e_planes = fine(s) ? 2 : 1;
    k.tn = p.Np / p.tile;
    k.alpha = 1.f / SCALE_P;
    k.beta = a;
    k.out = X;
    k.out_plane = p.x;
    k.out_batch = xb;
    k.turned = next;
    k.turned_plane = p.xt;
    k.turned_batch = xb;
    k.turned_planes = fine(s + 1) ? 2 : 1;
    k.result = x;
    k.rows = p.M;
    k.cols = p.N;
    k.result_turned = tall;
    const int rc = last ? launch_product<128, 128, 2, 2, PL, LAST, T>(k, batch, st)
                        : launch_product<128, 128, 2, 2, PL, PX, T>(k, batch, st);
    if (rc) return rc;
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

}  // namespace
}  // namespace xl

extern "C" size_t xl_newton_schulz_workspace_size(int64_t batch, int m, int n, int dtype) {
  using namespace xl;
  if (check_sizes("xl_newton_schulz_workspace_size", batch, m, n, dtype) || batch == 0 || m == 0 || n == 0) return 0;
  return plan_of(batch, m, n, dtype).bytes;
}

extern "C" int xl_newton_schulz(const void* g, void* x, int64_t batch, int m, int n, const float* coefficients, int steps,
                                float eps, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace xl;
  clear_error();
  const char* who = "xl_newton_schulz";
  if (const int rc = check_sizes(who, batch, m, n, dtype)) return rc;
  if (steps < 1 || !coefficients) return set_error(XL_ERR_INVALID_ARG, "%s: steps=%d (at least 1, with coefficients)", who, steps);
  if (!(eps >= 0.f)) return set_error(XL_ERR_INVALID_ARG, "%s: eps=%g (not negative)", who, (double)eps);
  // singular values start in [0, 1]: the most that a step's polynomial makes of them
  double most = 1.0;
  for (int s = 0; s < steps; ++s) {
    const double a = coefficients[3 * s], b = coefficients[3 * s + 1], c = coefficients[3 * s + 2], x2 = most * most;
    const double in_p = fabs(b) * x2 + fabs(c) * x2 * x2;
    double next = 0.0;
    for (int i = 0; i <= 1024; ++i) {
      const double v = most * i / 1024, y = fabs(v * (a + b * v * v + c * v * v * v * v));
      if (!(y <= next)) next = y;
    }
    if (!(in_p <= MOST_P) || !(next <= 0.99 * MOST_X))
      return set_error(XL_ERR_INVALID_ARG, "%s: step %d's coefficients (%g, %g, %g) take singular values out of range", who, s, a,
                       b, c);
    most = next * 1.01;  // between the samples, and the products' rounding
  }
  if (batch == 0 || m == 0 || n == 0) return XL_OK;
  if (!g || !x) return set_error(XL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (g == x) return set_error(XL_ERR_INVALID_ARG, "%s: x must not alias g", who);
  const Plan p = plan_of(batch, m, n, dtype);
  if (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255u))
    return set_error(XL_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", who, p.bytes,
                     workspace_bytes);
  char* ws = (char*)workspace;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case XL_DTYPE_F32: return run<float, 2>(g, x, batch, m, n, coefficients, steps, eps, p, ws, st);
    case XL_DTYPE_BF16: return run<bf16_t, 1>(g, x, batch, m, n, coefficients, steps, eps, p, ws, st);
    default: return run<f16_t, 2>(g, x, batch, m, n, coefficients, steps, eps, p, ws, st);
  }
}
