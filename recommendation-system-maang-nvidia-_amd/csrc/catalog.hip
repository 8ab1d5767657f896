// catalog.hip — softmax cross entropy of N rows over a whole catalogue of V items, with its gradient,
// the logits never stored (the full-catalogue form of the in-batch retrieval loss of inbatch.hip,
// src/models.py:116,137 of the reference: there the vocabulary is the batch's own items).
//
//   s_nv = c <x_n, w_v>,  row_n = log sum_v exp s_nv - s_n,y,  loss = sum_n a_n row_n / Z
//   dx_n = (g/Z) c a_n (sum_v p_nv w_v - w_y),  dw_v = (g/Z) c sum_n a_n (p_nv - [v = y_n]) x_n
//
// One kernel form, cs_pass_kernel, serves both directions. A workgroup owns "resident" rows (held in
// registers as the matrix instructions' B operand) and streams the other matrix through LDS in tiles:
// S^T = T R^T, then exponentials in the accumulators, which are already the B operand of the second
// product O^T = T^T P^T, so neither S nor P leaves the registers. Row pass: R = x, T = w, a running
// maximum and sum, O = sum_v exp(s_v - m) w_v. Column pass: R = w, T = x, p from the row pass's lse,
// O = sum_n a_n p_nv x_n = dw. 4 N V D flops each (2 N V D for the row pass of an evaluation).
//
// The label's own term stays out of the row pass's sum. With o = log sum_{v != y} exp s_v and
// t = o - s_y the loss is log1p(exp t), 1 - p_y = sigmoid(t) = q and dx = q (O / l - w_y): no
// difference of nearly equal numbers where the label is nearly certain. The column pass takes -q for
// the label's element.
//
// bf16 inputs: one bf16 product, p rounded to bf16 (2^-8 of each term, as its output is). fp32 inputs:
// every operand as two fp16 terms h + l of the value scaled by a power of two (|x - h - l| <= 2^-22
// |x|, or 2^-39 of the scale's largest value), three products h h, h l, l h per fp32 product: half the
// matrix work of the exact three-term bf16 split, rounding below an fp32 dot product's own. Rows of x
// have a scale each; w, which the row pass sums over, has one. p is scaled against the running maximum
// (kept in both passes) so that unlikely items keep their relative precision, and each tile's sum
// is formed in fresh accumulators and added in fp32 (the matrix unit's long running sums lose bits).
#include "split.hpp"

#include <cfloat>
#include <cmath>

namespace rs {
namespace {

typedef _Float16 cs_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 cs_h2 __attribute__((ext_vector_type(2)));

constexpr float CS_MIN = -1e30f;     // the running maximum before any item
constexpr float CS_PS = 15.f;        // fp16 exponentials are formed at 2^15 (below 65504)
constexpr int CS_AMAX_BLOCKS = 512;  // partial maxima of |w|
constexpr double CS_LOG2E = 1.4426950408889634074;
constexpr double CS_LN2 = 0.69314718055994530942;

// device scalars of a call (in the kept buffer)
struct CsScal {
  float w_inv;   // 2^-e of the catalogue's scale (fp32), 1 (bf16)
  float c0;      // -exponent of the largest |a_n| / x-scale (fp32): keeps p a in fp16's range
  float inv_z;   // 1 / Z of the reduction
};

// row statistics the column pass streams beside x: per 32 rows four arrays of 32 words
enum { CS_LSE2 = 0, CS_COEF = 1, CS_KX = 2, CS_LAB = 3 };
__host__ __device__ inline int64_t cs_stat(int64_t n, int a) { return (n >> 5) * 128 + a * 32 + (n & 31); }

struct CsPass {
  const char* R;          // resident rows [nR][D] (plane stride r_plane bytes)
  const char* T;          // streamed rows [nT][D]
  int64_t nR, nT, t_last; // valid rows; the last streamed row that may be read
  int64_t r_plane, t_plane;
  int64_t tiles, per;     // streamed tiles, tiles per split
  int nrb;                // resident blocks
  const CsScal* scal;
  float scale, kbase;     // c, c log2 e
  const float* kx;        // row pass, fp32: 2^-e of each resident row
  const int32_t* lab;     // row pass: label of each resident row (< 0: none)
  const float* stat;      // column pass: statistics of the streamed rows
  const float* lq;        // column pass: log2 q of the streamed rows
  float *m, *l, *O;       // partials [split][nR](, [D])
  // column pass, one split: the gradient itself
  void* out;
  int64_t ld;             // its row length (0: partials)
  int out_bf16;
  const float* gscale;
};

template <int NP>
__device__ __forceinline__ f32x4 cs_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (NP == 1) return mfma16_bf16(a, b, c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(cs_h8, a), __builtin_bit_cast(cs_h8, b), c, 0, 0, 0);
}

// 16-B chunk ch of tile row r lies at chunk ch ^ cs_swz(r) of its LDS row: both the row reads (16 rows
// 8 a + b + const, one chunk each) and the transposed reads (16 rows, one chunk pair) then touch every
// bank evenly; bit 2 of the row does not enter, so rows r and r + 4 differ by an immediate.
template <int D>
__device__ __forceinline__ int cs_swz(int r) {
  if constexpr (D == 64) return (((r >> 1) & 1) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
  else return ((r & 3) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
}

// 16 B per lane from global memory to LDS at dst + 16 lane (dst uniform); only an explicit vmcnt waits
// for it
__device__ __forceinline__ void cs_glds16(const char* g, uint32_t dst) {
  const uint32_t m0v = __builtin_amdgcn_readfirstlane(dst);
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(g), "s"(m0v)
               : "memory");
}

template <typename T>
__device__ __forceinline__ T cs_lds(uint32_t off) {
  return *reinterpret_cast<__attribute__((address_space(3))) const T*>(off);
}

// workgroup id -> a permutation in which consecutive ids share an XCD (workgroups go round the 8
// XCDs), so that the blocks streaming one range read it from one L2
__device__ __forceinline__ int cs_xcd(int id, int n) {
  const int per = n / 8, rem = n % 8, x = id & 7, j = id >> 3;
  return x * per + (x < rem ? x : rem) + j;
}

enum { CS_STATS = 0, CS_ROW = 1, CS_COL = 2 };

// Register and LDS budget: 8 waves of 32 resident rows (two per SIMD, 256 registers) up to D = 128;
// D = 256 fp32 holds x's two planes and O in 512 registers, one wave per SIMD.
constexpr int cs_waves(int D) { return D == 256 ? 4 : 8; }
constexpr int CS_UB = 2;   // 16-row subtiles of resident rows per wave
constexpr int CS_KT = 64;  // streamed rows per tile
constexpr int cs_block_rows(int D) { return 16 * CS_UB * cs_waves(D); }

template <int D, int NP, int MODE>
__global__ __launch_bounds__(64 * cs_waves(D), cs_waves(D) / 4) void cs_pass_kernel(CsPass p) {
  constexpr int UB = CS_UB, NW = cs_waves(D), KT = CS_KT;
  constexpr int CH = D / 8, ROWB = 2 * D, PLANE = KT * ROWB, IMG = NP * PLANE, NS = KT / 32, NDT = D / 16, NC = D / 32;
  constexpr int STAT = MODE == CS_COL ? KT * 16 : 0;
  constexpr bool RUNMAX = MODE != CS_COL || NP == 2;
  __shared__ __attribute__((aligned(1024))) char smem[2 * (IMG + STAT)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, i16 = lane & 15;
  const int id = cs_xcd(blockIdx.x, gridDim.x);
  const int split = id / p.nrb;
  const int64_t r0 = (int64_t)(id % p.nrb) * cs_block_rows(D) + wave * (16 * UB);
  const int64_t tb0 = split * p.per, tb1 = tb0 + p.per < p.tiles ? tb0 + p.per : p.tiles;
  const uint32_t lds0 = (uint32_t) reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem);

  auto copy = [&](int64_t t, int buf) __attribute__((always_inline)) {
    const int64_t row0 = t * KT;
#pragma unroll
    for (int i = 0; i < PLANE / (NW * 1024); ++i) {
      const int row = i * (NW * 64 / CH) + tid / CH;
      const int ch = (tid % CH) ^ cs_swz<D>(row);
      const int64_t rr = row0 + row < p.t_last ? row0 + row : p.t_last;
      const char* s = p.T + rr * ROWB + ch * 16;
#pragma unroll
      for (int pl = 0; pl < NP; ++pl)
        cs_glds16(s + pl * p.t_plane, lds0 + buf * (IMG + STAT) + pl * PLANE + i * NW * 1024 + wave * 1024);
    }
    if constexpr (MODE == CS_COL)
      if (wave == 0) cs_glds16((const char*)p.stat + row0 * 16 + lane * 16, lds0 + buf * (IMG + STAT) + IMG);
  };
  if (tb0 < tb1) copy(tb0, 0);

  // resident rows as the B operand: column i16 of subtile ub, k = 32 c + 8 g ..
  u32x4 xq[UB][NC][NP];
  float kq[UB];
  int32_t lab[UB];
#pragma unroll
  for (int ub = 0; ub < UB; ++ub) {
    int64_t q = r0 + 16 * ub + i16;
    q = q < p.nR ? q : p.nR - 1;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int pl = 0; pl < NP; ++pl)
        xq[ub][c][pl] = *reinterpret_cast<const u32x4*>(p.R + pl * p.r_plane + q * ROWB + (4 * c + g) * 16);
    if constexpr (MODE != CS_COL) {
      // FLT_MIN: a masked item's -inf must stay -inf after the product
      kq[ub] = NP == 2 ? fminf(fmaxf(p.kbase * p.scal->w_inv * p.kx[q], FLT_MIN), FLT_MAX) : p.kbase;
      lab[ub] = p.lab[q];
    }
  }
  const float kw = NP == 2 ? p.kbase * p.scal->w_inv : p.kbase;
  const float ps = NP == 2 ? (MODE == CS_COL ? CS_PS + p.scal->c0 : CS_PS) : 0.f;

  // row reads: A row i16 of subtile (s, kb) = tile row 32 s + 4 kb + 8 (i16 / 4) + i16 % 4, chunk 4 c + g
  uint32_t ab[NC < 4 ? NC : 4];
  {
    const int rho = 8 * (i16 >> 2) + (i16 & 3);
#pragma unroll
    for (int c = 0; c < (NC < 4 ? NC : 4); ++c) ab[c] = lds0 + rho * ROWB + (((4 * c + g) ^ cs_swz<D>(rho)) * 16);
  }
  // transposed reads: tile row 32 s + 8 g + 4 h + i16 / 4, columns 16 dt + 4 (i16 % 4) ..
  uint32_t tb[NDT < 8 ? NDT : 8];
  {
    const int rho = 8 * g + (i16 >> 2), pp = i16 & 3;
#pragma unroll
    for (int dt = 0; dt < (NDT < 8 ? NDT : 8); ++dt)
      tb[dt] = lds0 + rho * ROWB + (((2 * dt + (pp >> 1)) ^ cs_swz<D>(rho)) * 16) + 8 * (pp & 1);
  }

  f32x4 O[MODE == CS_STATS ? 1 : NDT][UB];
#pragma unroll
  for (int dt = 0; dt < (MODE == CS_STATS ? 1 : NDT); ++dt)
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) O[dt][ub] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m[UB], l[UB];  // the maximum of log2 terms, less ps; this lane's sum
#pragma unroll
  for (int ub = 0; ub < UB; ++ub) {
    m[ub] = CS_MIN;
    l[ub] = 0.f;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  for (int64_t t = tb0; t < tb1; ++t) {
    const int buf = (int)(t - tb0) & 1;
    const uint32_t bo = buf * (IMG + STAT);
    if (t + 1 < tb1) copy(t + 1, buf ^ 1);

    f32x4 s[2 * NS][UB];  // [2 sub + kb][ub]: streamed row 32 sub + 8 g + 4 kb + r, resident 16 ub + i16
#pragma unroll
    for (int k = 0; k < 2 * NS; ++k)
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) s[k][ub] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 2 * NS; ++k) {
        u32x4 a[NP];
#pragma unroll
        for (int pl = 0; pl < NP; ++pl)
          a[pl] = cs_lds<u32x4>(ab[c & 3] + bo + (c >> 2) * 256 + (32 * (k >> 1) + 4 * (k & 1)) * ROWB + pl * PLANE);
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
          if constexpr (NP == 2) {
            s[k][ub] = cs_mfma<NP>(a[1], xq[ub][c][0], s[k][ub]);
            s[k][ub] = cs_mfma<NP>(a[0], xq[ub][c][1], s[k][ub]);
          }
          s[k][ub] = cs_mfma<NP>(a[0], xq[ub][c][0], s[k][ub]);
        }
      }

    bool hit = false;  // a label's element lies in this tile (uniform)
    if constexpr (MODE == CS_COL) {
      // log2 p = s k_n - lse2_n
#pragma unroll
      for (int k = 0; k < 2 * NS; ++k) {
        const uint32_t sb = lds0 + bo + IMG + (k >> 1) * 512 + (8 * g + 4 * (k & 1)) * 4;
        const f32x4 ls = cs_lds<f32x4>(sb + CS_LSE2 * 128);
        f32x4 kn = f32x4{kw, kw, kw, kw};
        if constexpr (NP == 2) kn = cs_lds<f32x4>(sb + CS_KX * 128);
#pragma unroll
        for (int ub = 0; ub < UB; ++ub)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[k][ub][r] = __builtin_fmaf(s[k][ub][r], kn[r], -ls[r]);
      }
      const int32_t lb = cs_lds<int32_t>(lds0 + bo + IMG + (lane >> 5) * 512 + CS_LAB * 128 + (lane & 31) * 4);
      hit = __any((uint32_t)(lb - (int32_t)r0) < (uint32_t)(16 * UB));
      if (hit) {
#pragma unroll
        for (int k = 0; k < 2 * NS; ++k) {
          const int n4 = 8 * g + 4 * (k & 1);
          const int64_t row = t * KT + 32 * (k >> 1) + n4;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int32_t ln = cs_lds<int32_t>(lds0 + bo + IMG + (k >> 1) * 512 + CS_LAB * 128 + (n4 + r) * 4);
            const float lqn = p.lq[row + r];
#pragma unroll
            for (int ub = 0; ub < UB; ++ub)
              if (ln == (int32_t)r0 + 16 * ub + i16) s[k][ub][r] = lqn;
          }
        }
      }
    } else {
      const int64_t v0 = t * KT;
      bool mine = false;
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) mine |= (uint32_t)(lab[ub] - (int32_t)v0) < (uint32_t)KT;
      if (__any(mine) || v0 + KT > p.nT) {
#pragma unroll
        for (int k = 0; k < 2 * NS; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int64_t v = v0 + 32 * (k >> 1) + 8 * g + 4 * (k & 1) + r;
#pragma unroll
            for (int ub = 0; ub < UB; ++ub)
              if (v >= p.nT || (int32_t)v == lab[ub]) s[k][ub][r] = -INFINITY;
          }
      }
    }

    if constexpr (RUNMAX) {
      float mx[UB];
      bool up = false;
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) {
        mx[ub] = fmaxf(s[0][ub][0], s[0][ub][1]);
#pragma unroll
        for (int k = 0; k < 2 * NS; ++k)
#pragma unroll
          for (int r = k == 0 ? 2 : 0; r < 4; r += 2) mx[ub] = fmaxf(fmaxf(s[k][ub][r], s[k][ub][r + 1]), mx[ub]);
        mx[ub] = (MODE == CS_COL ? mx[ub] : mx[ub] * kq[ub]) - ps;
        up |= mx[ub] > m[ub];
      }
      if (__any(up)) {
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
          float x = fmaxf(mx[ub], __shfl_xor(mx[ub], 16, 64));
          x = fmaxf(x, __shfl_xor(x, 32, 64));
          x = fmaxf(x, m[ub]);
          const float al = __builtin_amdgcn_exp2f(m[ub] - x);
          m[ub] = x;
          l[ub] *= al;
          if constexpr (MODE != CS_STATS)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) O[dt][ub] *= al;
        }
      }
    }

    // exponentials; P's words are the second product's B operand: k = 8 g + j of sub = [2 sub][j], j < 4,
    // [2 sub + 1][j - 4]
    u32x4 pb[MODE == CS_STATS ? 1 : NS][UB][NP];
#pragma unroll
    for (int k = 0; k < 2 * NS; ++k) {
      f32x4 cf;
      if constexpr (MODE == CS_COL)
        cf = cs_lds<f32x4>(lds0 + bo + IMG + (k >> 1) * 512 + CS_COEF * 128 + (8 * g + 4 * (k & 1)) * 4);
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) {
        f32x4 e;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = s[k][ub][r];
          if constexpr (MODE != CS_COL) e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, kq[ub], -m[ub]));
          else if constexpr (NP == 2) e[r] = __builtin_amdgcn_exp2f(x - m[ub]) * cf[r];
          else e[r] = __builtin_amdgcn_exp2f(x) * cf[r];
        }
        if constexpr (MODE != CS_COL) l[ub] += (e[0] + e[1]) + (e[2] + e[3]);
        if constexpr (MODE == CS_COL)
          if (hit) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int32_t ln =
                  cs_lds<int32_t>(lds0 + bo + IMG + (k >> 1) * 512 + CS_LAB * 128 + (8 * g + 4 * (k & 1) + r) * 4);
              if (ln == (int32_t)r0 + 16 * ub + i16) e[r] = -e[r];
            }
          }
        if constexpr (MODE != CS_STATS) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float a = e[2 * h], b = e[2 * h + 1];
            if constexpr (NP == 1) pb[k >> 1][ub][0][2 * (k & 1) + h] = ib_pk(a, b);
            else {
              const cs_h2 hi = __builtin_bit_cast(cs_h2, __builtin_amdgcn_cvt_pkrtz(a, b));
              const cs_h2 lo = __builtin_bit_cast(cs_h2, __builtin_amdgcn_cvt_pkrtz(a - (float)hi[0], b - (float)hi[1]));
              pb[k >> 1][ub][0][2 * (k & 1) + h] = __builtin_bit_cast(uint32_t, hi);
              pb[k >> 1][ub][1][2 * (k & 1) + h] = __builtin_bit_cast(uint32_t, lo);
            }
          }
        }
      }
    }

    if constexpr (MODE != CS_STATS) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        f32x4 f[UB];
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) f[ub] = NP == 1 ? O[dt][ub] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) {
          u32x4 a[NP];
#pragma unroll
          for (int pl = 0; pl < NP; ++pl)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const ib_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) ib_s16x4*)(uintptr_t)(tb[dt & 7] + bo + (dt >> 3) * 256 +
                                                                (32 * sub + 4 * h) * ROWB + pl * PLANE));
              const u32x2 w2 = __builtin_bit_cast(u32x2, v);
              a[pl][2 * h] = w2[0];
              a[pl][2 * h + 1] = w2[1];
            }
#pragma unroll
          for (int ub = 0; ub < UB; ++ub) {
            if constexpr (NP == 2) {
              f[ub] = cs_mfma<NP>(a[1], pb[sub][ub][0], f[ub]);
              f[ub] = cs_mfma<NP>(a[0], pb[sub][ub][1], f[ub]);
            }
            f[ub] = cs_mfma<NP>(a[0], pb[sub][ub][0], f[ub]);
          }
        }
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) O[dt][ub] = NP == 1 ? f[ub] : O[dt][ub] + f[ub];
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

#pragma unroll
  for (int ub = 0; ub < UB; ++ub) {
    const int64_t q = r0 + 16 * ub + i16;
    float sum = l[ub];
    if constexpr (MODE != CS_COL) {
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
    }
    if (q >= p.nR) continue;
    if (MODE == CS_COL && p.ld) {
      // dw = O 2^m (the row scales are in the coefficients), times c g / Z
      float f = p.scale * p.scal->inv_z * (p.gscale ? *p.gscale : 1.f);
      if constexpr (NP == 2) f *= __builtin_amdgcn_exp2f(m[ub]);
#pragma unroll
      for (int dt = 0; dt < (MODE == CS_STATS ? 1 : NDT); ++dt) {
        const f32x4 v = O[dt][ub] * f;
        const int64_t d = 16 * dt + 4 * g;
        if (p.out_bf16) {
          __bf16* o = (__bf16*)p.out + q * p.ld + d;
          if (p.ld == D) *reinterpret_cast<u32x2*>(o) = u32x2{ib_pk(v[0], v[1]), ib_pk(v[2], v[3])};
          else
            for (int r = 0; r < 4; ++r)
              if (d + r < p.ld) o[r] = (__bf16)v[r];
        } else {
          float* o = (float*)p.out + q * p.ld + d;
          if (p.ld == D) *reinterpret_cast<f32x4*>(o) = v;
          else
            for (int r = 0; r < 4; ++r)
              if (d + r < p.ld) o[r] = v[r];
        }
      }
      continue;
    }
    const int64_t o = split * p.nR + q;
    if (g == 0) {
      if constexpr (RUNMAX) p.m[o] = m[ub];
      if constexpr (MODE != CS_COL) p.l[o] = sum;
    }
    if constexpr (MODE != CS_STATS)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(p.O + o * D + 16 * dt + 4 * g) = O[dt][ub];
  }
}

// ---- operand images ------------------------------------------------------------------------------
__device__ __forceinline__ float cs_finite_abs(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.f;
}
__device__ __forceinline__ float cs_block_max(float v, float* sh) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (unsigned i = 1; i < blockDim.x / 64; ++i) v = fmaxf(v, sh[i]);
  return v;
}

// largest finite |w| of each workgroup's share
__global__ __launch_bounds__(256) void cs_amax_kernel(const float* __restrict__ w, int64_t n, float* __restrict__ part) {
  __shared__ float sh[4];
  float a = 0.f;
  const int64_t n4 = n / 4, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += step) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(w + 4 * i);
    a = fmaxf(fmaxf(fmaxf(cs_finite_abs(v[0]), cs_finite_abs(v[1])), fmaxf(cs_finite_abs(v[2]), cs_finite_abs(v[3]))), a);
  }
  if (blockIdx.x == 0 && threadIdx.x < n - 4 * n4) a = fmaxf(a, cs_finite_abs(w[4 * n4 + threadIdx.x]));
  a = cs_block_max(a, sh);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// the power of two that brings a into [2^13, 2^14)
__device__ __forceinline__ int cs_exp(float a) {
  if (!(a > 0.f)) return 0;
  int e;
  (void)frexpf(a, &e);  // a in [2^(e-1), 2^e)
  const int k = 14 - e;
  return k < -100 ? -100 : k > 100 ? 100 : k;
}

struct CsImage {
  const void *x, *w;
  char *ximg, *wimg;       // wimg null: w is read as it is
  int64_t N, Npad, V, D;
  int64_t xplane, wplane;
  int64_t ignore;
  const int64_t* labels;
  int32_t* lab;
  float* kx;
  const float* part;
  CsScal* scal;
  int xblocks;
};

// x [N, D] and w [V, D] into padded 16-bit rows: two fp16 planes of the scaled values (fp32), a copy
// (bf16). A row of x whose label is the ignored one keeps its finite entries only (its weight in the
// column pass is zero, and zero times infinity would not be). 4 columns per lane.
template <int DP, int NP>
__global__ __launch_bounds__(256) void cs_image_kernel(CsImage p) {
  constexpr int LPR = DP / 4, RPB = 256 / LPR;  // lanes per row, rows per workgroup
  __shared__ float sh[4];
  const int c = (threadIdx.x % LPR) * 4, rr = threadIdx.x / LPR;
  const bool is_x = (int)blockIdx.x < p.xblocks;
  float wscale = 1.f;
  if (NP == 2 && !is_x) {
    float a = 0.f;
    for (int i = threadIdx.x; i < CS_AMAX_BLOCKS; i += 256) a = fmaxf(a, p.part[i]);
    const int e = cs_exp(cs_block_max(a, sh));
    wscale = ldexpf(1.f, e);
    if ((int)blockIdx.x == p.xblocks && threadIdx.x == 0) p.scal->w_inv = ldexpf(1.f, -e);
  }
  const int64_t blk = is_x ? blockIdx.x : blockIdx.x - p.xblocks;
  const int64_t nblk = is_x ? p.xblocks : gridDim.x - p.xblocks;
  const int64_t rows = is_x ? p.N : p.V, rows_pad = is_x ? p.Npad : p.V;
  const void* src = is_x ? p.x : p.w;
  char* dst = is_x ? p.ximg : p.wimg;
  const int64_t plane = is_x ? p.xplane : p.wplane;
  const bool vec = p.D % 4 == 0;
  for (int64_t r = blk * RPB + rr; r < rows_pad; r += nblk * RPB) {
    int32_t lb = -1;
    if (is_x) {
      if (r < rows) {
        const int64_t y = p.labels[r];
        lb = y == p.ignore ? -1 : (y >= 0 && y < p.V) ? (int32_t)y : -2;
      }
      if (c == 0) p.lab[r] = lb;
    }
    if constexpr (NP == 1) {
      const uint16_t* s = (const uint16_t*)src + r * p.D + c;
      uint16_t h[4] = {0, 0, 0, 0};
      if (r < rows)
        for (int j = 0; j < 4; ++j)
          if (c + j < p.D) {
            h[j] = s[j];
            if (is_x && lb < 0 && (h[j] & 0x7f80) == 0x7f80) h[j] = 0;
          }
      *reinterpret_cast<u32x2*>(dst + r * (2 * DP) + 2 * c) =
          u32x2{h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16)};
    } else {
      const float* s = (const float*)src + r * p.D + c;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (r < rows) {
        if (vec) {
          if (c < p.D) v = *reinterpret_cast<const f32x4*>(s);
        } else {
          for (int j = 0; j < 4; ++j)
            if (c + j < p.D) v[j] = s[j];
        }
      }
      float sc = wscale;
      if (is_x) {
        if (lb < 0)
          for (int j = 0; j < 4; ++j) v[j] = fabsf(v[j]) <= FLT_MAX ? v[j] : 0.f;
        float a = fmaxf(fmaxf(cs_finite_abs(v[0]), cs_finite_abs(v[1])), fmaxf(cs_finite_abs(v[2]), cs_finite_abs(v[3])));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
        const int e = cs_exp(a);
        sc = ldexpf(1.f, e);
        if (c == 0) p.kx[r] = ldexpf(1.f, -e);
      }
      uint32_t h[2], lo[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float a = v[2 * j] * sc, b = v[2 * j + 1] * sc;
        const cs_h2 hh = {(_Float16)a, (_Float16)b};
        const cs_h2 ll = {(_Float16)(a - (float)hh[0]), (_Float16)(b - (float)hh[1])};
        h[j] = __builtin_bit_cast(uint32_t, hh);
        lo[j] = __builtin_bit_cast(uint32_t, ll);
      }
      *reinterpret_cast<u32x2*>(dst + r * (2 * DP) + 2 * c) = u32x2{h[0], h[1]};
      *reinterpret_cast<u32x2*>(dst + plane + r * (2 * DP) + 2 * c) = u32x2{lo[0], lo[1]};
    }
  }
}

// ---- rows of the forward -------------------------------------------------------------------------
struct CsRows {
  const void *x, *w;
  int bf16;
  int64_t N, Npad, V, D;
  int nsplit;
  const float *m, *l, *O;
  const int32_t* lab;
  const float* weights;
  const float* kx;
  const CsScal* scal;
  float scale, kbase;
  float *row, *lse, *dx, *stat, *lq;
};
__device__ __forceinline__ float cs_ld(const void* x, int bf16, int64_t i) {
  return bf16 ? (float)((const __bf16*)x)[i] : ((const float*)x)[i];
}

// one wave per row: joins the splits, the label's logit (64-bit sums), the row's loss, its statistics
// for the column pass and its unit gradient a q (O / l - w_y)
template <int DP, int NP>
__global__ __launch_bounds__(256) void cs_rows_kernel(CsRows p) {
  constexpr int VEC = DP / 64;
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= p.Npad) return;
  const float kw = NP == 2 ? p.kbase * p.scal->w_inv : p.kbase;
  if (n >= p.N) {
    if (lane == 0) {
      p.stat[cs_stat(n, CS_LSE2)] = INFINITY;
      p.stat[cs_stat(n, CS_COEF)] = 0.f;
      p.stat[cs_stat(n, CS_KX)] = kw;
      reinterpret_cast<int32_t*>(p.stat)[cs_stat(n, CS_LAB)] = -1;
      p.lq[n] = 0.f;
    }
    return;
  }
  const int32_t lb = p.lab[n];
  float M = CS_MIN;
  for (int s = lane; s < p.nsplit; s += 64) M = fmaxf(M, p.m[s * p.N + n]);
  M = wave_max(M);
  double L = 0.;
  for (int s = lane; s < p.nsplit; s += 64) {
    const float mv = p.m[s * p.N + n];
    L += (double)p.l[s * p.N + n] * (double)__builtin_amdgcn_exp2f(mv - M);
  }
  L = wave_sum_d(L);
  // in log2 units: the other items' log sum and the label's logit
  const double o2 = L == 0. ? -INFINITY : (double)M + log2(L);
  double sy = 0.;
  if (lb >= 0) {
    for (int64_t d = lane; d < p.D; d += 64)
      sy += (double)cs_ld(p.x, p.bf16, n * p.D + d) * (double)cs_ld(p.w, p.bf16, (int64_t)lb * p.D + d);
    sy = wave_sum_d(sy) * (double)p.scale * CS_LOG2E;
  }
  const float a = p.weights ? p.weights[n] : 1.f;
  const float t = (float)((o2 - sy) * CS_LN2);
  const float et = expf(-fabsf(t)), soft = log1pf(et);
  const float q = t > 0.f ? 1.f / (1.f + et) : et / (1.f + et);  // NaN stays NaN
  const double lse2 = lb >= 0 ? fmax(o2, sy) + (double)soft * CS_LOG2E : o2;
  if (lane == 0) {
    p.row[n] = lb >= 0 ? soft + fmaxf(t, 0.f) : lb == -1 ? 0.f : NAN;
    p.lse[n] = (float)(lse2 * CS_LN2);
    const bool live = lb >= 0;
    float coef = live ? a : 0.f;
    if (NP == 2) coef *= p.kx[n];
    // NaN statistics of a labelled row reach every item's gradient, as the formula's do
    p.stat[cs_stat(n, CS_LSE2)] = live ? (float)lse2 : INFINITY;
    p.stat[cs_stat(n, CS_COEF)] = coef;
    p.stat[cs_stat(n, CS_KX)] = NP == 2 ? fminf(fmaxf(kw * p.kx[n], FLT_MIN), FLT_MAX) : kw;
    reinterpret_cast<int32_t*>(p.stat)[cs_stat(n, CS_LAB)] = lb;
    p.lq[n] = (float)(o2 - lse2);
  }
  if (!p.dx) return;
  float o[VEC] = {};
  if (lb >= 0) {
    for (int s = 0; s < p.nsplit; ++s) {
      const float f = __builtin_amdgcn_exp2f(p.m[s * p.N + n] - M);
      const float* os = p.O + (s * p.N + n) * DP + lane * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] += f * os[j];
    }
  }
  const float il = L == 0. ? 0.f : (float)((NP == 2 ? (double)p.scal->w_inv : 1.) / L);
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const int64_t d = lane * VEC + j;
    if (d >= p.D) continue;
    float v = 0.f;
    if (lb >= 0) v = L == 0. ? 0.f : a * q * (o[j] * il - cs_ld(p.w, p.bf16, (int64_t)lb * p.D + d));
    else if (lb == -2) v = NAN;
    p.dx[n * p.D + d] = v;
  }
}

// the loss, 1 / Z and the coefficients' exponent; one workgroup, fixed order
__global__ __launch_bounds__(1024) void cs_total_kernel(const float* __restrict__ row, const int32_t* __restrict__ lab,
                                                         const float* __restrict__ weights, const float* __restrict__ stat,
                                                         int64_t N, int mean, CsScal* scal, float* __restrict__ loss) {
  __shared__ double sh[2][16];
  __shared__ float shm[16];
  double s = 0., z = 0.;
  float cm = 0.f;
  for (int64_t n = threadIdx.x; n < N; n += 1024) {
    const int32_t lb = lab[n];
    if (lb == -1) continue;
    const float a = weights ? weights[n] : 1.f;
    s += (double)a * (double)row[n];
    z += (double)a;
    cm = fmaxf(cm, cs_finite_abs(stat[cs_stat(n, CS_COEF)]));
  }
  s = wave_sum_d(s);
  z = wave_sum_d(z);
  cm = wave_max(cm);
  if ((threadIdx.x & 63) == 0) {
    sh[0][threadIdx.x >> 6] = s;
    sh[1][threadIdx.x >> 6] = z;
    shm[threadIdx.x >> 6] = cm;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = z = 0.;
    cm = 0.f;
    for (int i = 0; i < 16; ++i) {
      s += sh[0][i];
      z += sh[1][i];
      cm = fmaxf(cm, shm[i]);
    }
    const double inv = !mean ? 1. : z != 0. ? 1. / z : 0.;
    int e = 0;
    if (cm > 0.f) (void)frexpf(cm, &e);  // cm < 2^e
    scal->c0 = (float)-e;
    scal->inv_z = (float)inv;
    *loss = (float)(s * inv);
  }
}

// ---- backward ------------------------------------------------------------------------------------
// dx = c g / Z times the forward's unit gradient
__global__ __launch_bounds__(256) void cs_dx_kernel(const float* __restrict__ u, int64_t n, float scale,
                                                    const CsScal* __restrict__ scal, const float* __restrict__ gscale,
                                                    void* __restrict__ out, int bf16) {
  const float f = scale * scal->inv_z * (gscale ? *gscale : 1.f);
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i + 4 <= n) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(u + i) * f;
    if (bf16) *reinterpret_cast<u32x2*>((__bf16*)out + i) = u32x2{ib_pk(v[0], v[1]), ib_pk(v[2], v[3])};
    else *reinterpret_cast<f32x4*>((float*)out + i) = v;
  } else {
    for (int64_t j = i; j < n; ++j) {
      if (bf16) ((__bf16*)out)[j] = (__bf16)(u[j] * f);
      else ((float*)out)[j] = u[j] * f;
    }
  }
}

// dw from the column pass's partials of several row ranges, in their order
template <int DP, int NP>
__global__ __launch_bounds__(256) void cs_dw_kernel(const float* __restrict__ m, const float* __restrict__ O, int nsplit,
                                                    int64_t V, int64_t D, float scale, const CsScal* __restrict__ scal,
                                                    const float* __restrict__ gscale, void* __restrict__ out, int bf16) {
  constexpr int LPR = DP / 4, RPB = 256 / LPR;
  const int c = (threadIdx.x % LPR) * 4;
  const int64_t v = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  if (v >= V) return;
  float M = CS_MIN;
  if constexpr (NP == 2)
    for (int s = 0; s < nsplit; ++s) M = fmaxf(M, m[s * V + v]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < nsplit; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(O + (s * V + v) * DP + c);
    if constexpr (NP == 2) o += x * __builtin_amdgcn_exp2f(m[s * V + v] - M);
    else o += x;
  }
  float f = scale * scal->inv_z * (gscale ? *gscale : 1.f);
  if constexpr (NP == 2) f *= __builtin_amdgcn_exp2f(M);
  for (int j = 0; j < 4; ++j)
    if (c + j < D) {
      if (bf16) ((__bf16*)out)[v * D + c + j] = (__bf16)(o[j] * f);
      else ((float*)out)[v * D + c + j] = o[j] * f;
    }
}

// ---- host ----------------------------------------------------------------------------------------
int cs_width(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Streamed ranges per resident block. Workgroups run one per CU (256 slots); a range costs its tiles
// plus a fixed start-up and join of about 4 tiles, so the split that needs the fewest tile times wins.
int cs_nsplit(int64_t nrb, int64_t tiles) {
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int64_t s = 1; s <= tiles && s <= 1024 && (s == 1 || nrb * s <= 2048); ++s) {
    const int64_t per = ceil_div(tiles, s);
    if (ceil_div(tiles, per) != s) continue;
    const int64_t cost = ceil_div(nrb * s, 256) * (per + 4) + s / 16;
    if (cost < best_cost) {
      best_cost = cost;
      best = (int)s;
    }
  }
  return best;
}

struct CsShape {
  int64_t N, Npad, V, D;
  int DP, NP, es;
  bool wimage;
  int rsplit, csplit;
  int64_t rtiles, rper, ctiles, cper, rnrb, cnrb;
};
CsShape cs_shape(int64_t N, int64_t V, int64_t D, int dtype) {
  CsShape s;
  s.N = N;
  s.V = V;
  s.D = D;
  s.DP = cs_width(D);
  s.NP = dtype == RS_DTYPE_F32 ? 2 : 1;
  s.es = dtype == RS_DTYPE_F32 ? 4 : 2;
  s.Npad = (N + 63) / 64 * 64;
  s.wimage = s.NP == 2 || D != s.DP;
  const int rows = cs_block_rows(s.DP);
  s.rtiles = ceil_div(V, 64);
  s.ctiles = s.Npad / 64;
  s.rnrb = ceil_div(N, rows);
  s.cnrb = ceil_div(V, rows);
  s.rsplit = N ? cs_nsplit(s.rnrb, s.rtiles) : 1;
  s.csplit = s.ctiles ? cs_nsplit(s.cnrb, s.ctiles) : 1;
  s.rper = ceil_div(s.rtiles, s.rsplit);
  s.cper = s.ctiles ? ceil_div(s.ctiles, s.csplit) : 1;
  return s;
}

struct CsKeep {
  CsScal* scal;
  char *ximg, *wimg;
  int32_t* lab;
  float *kx, *stat, *lq, *dx;
  bool ok;
  size_t bytes;
  CsKeep(void* base, size_t size, const CsShape& s, int want) {
    Carve c(base, size);
    scal = c.take<CsScal>(1);
    ximg = c.take<char>((size_t)s.Npad * s.DP * 2 * s.NP);
    wimg = s.wimage ? c.take<char>((size_t)s.V * s.DP * 2 * s.NP) : nullptr;
    lab = c.take<int32_t>(s.Npad);
    kx = c.take<float>(s.Npad);
    stat = c.take<float>(s.Npad * 4);
    lq = c.take<float>(s.Npad);
    dx = want & RS_CATALOG_DX ? c.take<float>((size_t)s.N * s.D) : nullptr;
    bytes = align_up(c.off, 256);
    ok = c.ok();
  }
};
struct CsFwdWs {
  float *part, *m, *l, *O;
  bool ok;
  size_t bytes;
  CsFwdWs(void* base, size_t size, const CsShape& s, int want) {
    Carve c(base, size);
    part = c.take<float>(CS_AMAX_BLOCKS);
    m = c.take<float>((size_t)s.rsplit * s.N);
    l = c.take<float>((size_t)s.rsplit * s.N);
    O = want & RS_CATALOG_DX ? c.take<float>((size_t)s.rsplit * s.N * s.DP) : nullptr;
    bytes = align_up(c.off, 256);
    ok = c.ok();
  }
};
struct CsBwdWs {
  float *m, *O;
  bool ok;
  size_t bytes;
  CsBwdWs(void* base, size_t size, const CsShape& s, int want) {
    Carve c(base, size);
    const bool part = (want & RS_CATALOG_DW) && s.csplit > 1;
    m = part ? c.take<float>((size_t)s.csplit * s.V) : nullptr;
    O = part ? c.take<float>((size_t)s.csplit * s.V * s.DP) : nullptr;
    bytes = align_up(c.off, 256);
    ok = c.ok();
  }
};

template <int MODE>
void cs_launch_pass(const CsShape& s, const CsPass& p, int64_t grid, hipStream_t st) {
#define CS_GO(WD, PL) \
  if (s.DP == WD && s.NP == PL) \
    hipLaunchKernelGGL((cs_pass_kernel<WD, PL, MODE>), dim3((unsigned)grid), dim3(64 * cs_waves(WD)), 0, st, p);
  CS_GO(64, 1) CS_GO(64, 2) CS_GO(128, 1) CS_GO(128, 2) CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
}

int cs_check(int64_t N, int64_t V, int64_t D, int dtype, float scale, int want, const char* what) {
  RS_REQUIRE(N >= 0 && V >= 1 && D >= 1, "%s: bad sizes N=%lld V=%lld D=%lld", what, (long long)N, (long long)V,
             (long long)D);
  RS_REQUIRE(N < (1ll << 30) && V < (1ll << 30), "%s: N and V must be below 2^30", what);
  RS_REQUIRE(dtype == RS_DTYPE_F32 || dtype == RS_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
  RS_REQUIRE(scale > 0.f && scale <= FLT_MAX, "%s: scale must be positive and finite", what);
  RS_REQUIRE((want & ~(RS_CATALOG_DX | RS_CATALOG_DW)) == 0, "%s: unknown gradient flags %d", what, want);
  if (D > 256) {
    set_error("%s: width %lld is above 256", what, (long long)D);
    return RS_ERR_UNSUPPORTED;
  }
  return RS_OK;
}

}  // namespace
}  // namespace rs

using namespace rs;

extern "C" size_t rs_catalog_softmax_keep_bytes(int64_t N, int64_t V, int64_t D, int dtype, int want) {
  if (cs_check(N, V, D, dtype, 1.f, want, "catalog_softmax") != RS_OK) return 0;
  return CsKeep(nullptr, 0, cs_shape(N, V, D, dtype), want).bytes;
}

extern "C" size_t rs_catalog_softmax_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype, int want) {
  if (cs_check(N, V, D, dtype, 1.f, want, "catalog_softmax") != RS_OK) return 0;
  const CsShape s = cs_shape(N, V, D, dtype);
  const size_t a = CsFwdWs(nullptr, 0, s, want).bytes, b = CsBwdWs(nullptr, 0, s, want).bytes;
  return a > b ? a : b;
}

extern "C" int rs_catalog_softmax_fwd(const void* X, const void* W, const int64_t* labels, const float* weights,
                                      int64_t N, int64_t V, int64_t D, int dtype, float scale, int64_t ignore_index,
                                      int mean, int want, float* loss, float* row_loss, float* lse, void* keep,
                                      size_t keep_bytes, void* workspace, size_t workspace_bytes, rs_stream_t stream) {
  const int rc = cs_check(N, V, D, dtype, scale, want, "catalog_softmax_fwd");
  if (rc != RS_OK) return rc;
  RS_REQUIRE(W && loss && keep && workspace && (N == 0 || (X && labels && row_loss && lse)),
             "catalog_softmax_fwd: null pointer");
  RS_REQUIRE(aligned16(X) && aligned16(W) && aligned16(keep) && aligned16(workspace),
             "catalog_softmax_fwd: X, W, keep and workspace must be 16-byte aligned");
  const CsShape s = cs_shape(N, V, D, dtype);
  const CsKeep k(keep, keep_bytes, s, want);
  const CsFwdWs w(workspace, workspace_bytes, s, want);
  if (!k.ok || !w.ok) {
    set_error("catalog_softmax_fwd: %s too small", k.ok ? "workspace" : "keep buffer");
    return RS_ERR_WORKSPACE;
  }
  hipStream_t st = as_stream(stream);
  if (N > 0) {
    if (s.NP == 2) hipLaunchKernelGGL(cs_amax_kernel, dim3(CS_AMAX_BLOCKS), dim3(256), 0, st, (const float*)W, V * D, w.part);
    const int rpb = 256 / (s.DP / 4);
    CsImage im{X,    W,    k.ximg, k.wimg, N, s.Npad, V, D, s.Npad * s.DP * 2, V * s.DP * 2, ignore_index, labels, k.lab,
               k.kx, w.part, k.scal, 0};
    int64_t xb = ceil_div(s.Npad, rpb), wb = s.wimage ? ceil_div(V, rpb) : 0;
    im.xblocks = (int)(xb < 2048 ? xb : 2048);
    if (wb > 4096) wb = 4096;
    const dim3 gi((unsigned)(im.xblocks + wb));
#define CS_GO(WD, PL) \
  if (s.DP == WD && s.NP == PL) hipLaunchKernelGGL((cs_image_kernel<WD, PL>), gi, dim3(256), 0, st, im);
    CS_GO(64, 1) CS_GO(64, 2) CS_GO(128, 1) CS_GO(128, 2) CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
    CsPass p{};
    p.R = k.ximg;
    p.T = s.wimage ? k.wimg : (const char*)W;
    p.nR = N;
    p.nT = V;
    p.t_last = V - 1;
    p.r_plane = s.Npad * s.DP * 2;
    p.t_plane = V * s.DP * 2;
    p.tiles = s.rtiles;
    p.per = s.rper;
    p.nrb = (int)s.rnrb;
    p.scal = k.scal;
    p.scale = scale;
    p.kbase = (float)((double)scale * CS_LOG2E);
    p.kx = k.kx;
    p.lab = k.lab;
    p.m = w.m;
    p.l = w.l;
    p.O = w.O;
    if (want & RS_CATALOG_DX) cs_launch_pass<CS_ROW>(s, p, s.rnrb * s.rsplit, st);
    else cs_launch_pass<CS_STATS>(s, p, s.rnrb * s.rsplit, st);
    CsRows r{X, W, s.NP == 1, N, s.Npad, V, D, s.rsplit, w.m, w.l, w.O, k.lab, weights, k.kx, k.scal, scale, p.kbase,
             row_loss, lse, k.dx, k.stat, k.lq};
    const dim3 gr((unsigned)(s.Npad / 4));
#define CS_GO(WD, PL) \
  if (s.DP == WD && s.NP == PL) hipLaunchKernelGGL((cs_rows_kernel<WD, PL>), gr, dim3(256), 0, st, r);
    CS_GO(64, 1) CS_GO(64, 2) CS_GO(128, 1) CS_GO(128, 2) CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
  }
  hipLaunchKernelGGL(cs_total_kernel, dim3(1), dim3(1024), 0, st, row_loss, k.lab, weights, k.stat, N, mean, k.scal, loss);
  return check_launch("catalog_softmax_fwd");
}

extern "C" int rs_catalog_softmax_bwd(const void* W, int64_t N, int64_t V, int64_t D, int dtype, float scale, int want,
                                      const float* gscale, const void* keep, size_t keep_bytes, void* dX, void* dW,
                                      void* workspace, size_t workspace_bytes, rs_stream_t stream) {
  const int rc = cs_check(N, V, D, dtype, scale, want, "catalog_softmax_bwd");
  if (rc != RS_OK) return rc;
  RS_REQUIRE(W && keep && workspace, "catalog_softmax_bwd: null pointer");
  RS_REQUIRE(!dX || (want & RS_CATALOG_DX), "catalog_softmax_bwd: dX needs a forward with RS_CATALOG_DX");
  RS_REQUIRE(!dW || (want & RS_CATALOG_DW), "catalog_softmax_bwd: dW needs a forward with RS_CATALOG_DW");
  RS_REQUIRE(aligned16(W) && aligned16(keep) && aligned16(workspace) && aligned16(dX) && aligned16(dW),
             "catalog_softmax_bwd: W, keep, workspace, dX and dW must be 16-byte aligned");
  const CsShape s = cs_shape(N, V, D, dtype);
  const CsKeep k(const_cast<void*>(keep), keep_bytes, s, want);
  const CsBwdWs w(workspace, workspace_bytes, s, want);
  if (!k.ok || !w.ok) {
    set_error("catalog_softmax_bwd: %s too small", k.ok ? "workspace" : "keep buffer");
    return RS_ERR_WORKSPACE;
  }
  hipStream_t st = as_stream(stream);
  if (dX && N > 0)
    hipLaunchKernelGGL(cs_dx_kernel, dim3((unsigned)ceil_div(N * D, 1024)), dim3(256), 0, st, k.dx, N * D, scale, k.scal,
                       gscale, dX, s.NP == 1);
  if (dW) {
    CsPass p{};
    p.R = s.wimage ? k.wimg : (const char*)W;
    p.T = k.ximg;
    p.nR = V;
    p.nT = N;
    p.t_last = s.Npad - 1;
    p.r_plane = V * s.DP * 2;
    p.t_plane = s.Npad * s.DP * 2;
    p.tiles = s.ctiles;
    p.per = s.cper;
    p.nrb = (int)s.cnrb;
    p.scal = k.scal;
    p.scale = scale;
    p.kbase = (float)((double)scale * CS_LOG2E);
    p.stat = k.stat;
    p.lq = k.lq;
    p.m = w.m;
    p.O = w.O;
    p.out = dW;
    p.ld = s.csplit == 1 ? D : 0;
    p.out_bf16 = s.NP == 1;
    p.gscale = gscale;
    cs_launch_pass<CS_COL>(s, p, s.cnrb * s.csplit, st);
    if (s.csplit > 1) {
      const dim3 gd((unsigned)ceil_div(V, 256 / (s.DP / 4)));
#define CS_GO(WD, PL)                                                                                              \
  if (s.DP == WD && s.NP == PL)                                                                                     \
    hipLaunchKernelGGL((cs_dw_kernel<WD, PL>), gd, dim3(256), 0, st, w.m, w.O, s.csplit, V, D, scale, k.scal, gscale, \
                       dW, s.NP == 1);
      CS_GO(64, 1) CS_GO(64, 2) CS_GO(128, 1) CS_GO(128, 2) CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
    }
  }
  return check_launch("catalog_softmax_bwd");
}
