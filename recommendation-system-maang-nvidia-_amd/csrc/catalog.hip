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
// bf16 inputs: one bf16 product, p rounded to bf16 (2^-8 of each term, as its output is; p in two terms would
// be half as much matrix work again in each pass). The label's term keeps fp32's precision: dx has w_y itself,
// the column pass a second product of what -q's rounding lost, in the groups of rows that hold a label of the
// wave's items (16384 x 1M x 128: one group in a thousand; 1021 x 50k x 96: 49 -> 54 us).
//
// fp32 inputs: every operand as two fp16 terms h + l of the value scaled by a power of two (|x - h - l| <=
// 2^-22 |x|, or 2^-39 of the scale's largest value), three products h h, h l, l h per fp32 product: half the
// matrix work of the exact three-term bf16 split. Every row of x and every item has a scale of its own, so an
// item takes no bits from another. A logit's error is c sum_d |x_d w_d| 2^-20, like an fp32 product's own
// rounding, plus c D 2^-30 max|x_n| max|w_v|: more than the former only where an entry 2^10 and more below its
// item's largest one meets an x that makes up for it. In both passes P carries the streamed row's scale and is
// itself scaled against a running maximum of the scaled terms, so that unlikely or small items keep their
// relative precision, and each tile's sum is formed in fresh accumulators and added in fp32 (the matrix unit's
// long running sums lose bits).
//
// Bound: the matrix cores' rate at the clock their load leaves (1.9 to 2.1 GHz; 52 to 68 % of the cycles
// busy), the exponentials' vector work beside them. 16384 x 1M x 128 bf16, a training step: 13.1 to 14.2 ms,
// 1.2 to 1.3 PFLOP/s of its 8 N V D flops (a large bf16 library product: 1.16); 8192 x 100k x 128 fp32:
// 2.0 ms, 420 TFLOP/s, three fp16 products each (a large fp32 library product: 0.154 PFLOP/s). Fewer than ~300 rows:
// the catalogue's bytes.
#include "split.hpp"

#include <cfloat>
#include <cmath>

namespace rs {
namespace {

typedef _Float16 cs_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 cs_h2 __attribute__((ext_vector_type(2)));

constexpr float CS_MIN = -1e30f;     // the running maximum before any item
constexpr float CS_PS = 15.f;        // fp16 exponentials are formed at 2^15 (below 65504)
constexpr double CS_LOG2E = 1.4426950408889634074;
constexpr double CS_LN2 = 0.69314718055994530942;

// device scalars of a call (in the kept buffer)
struct CsScal {
  float inv_z;   // 1 / Z of the reduction
  int32_t neg;   // a labelled row's weight is negative
  float pad[2];
  float zero[4];  // 16 zero bytes, for the columns past a width
};

// Row statistics the column pass streams beside x, per 32 rows four arrays of 32 words: lse - log |a| in
// log2 units (infinite where the row takes no part), the factor of its scores, twice its label plus one for
// a negative weight (negative: no label), log2 (|a| q). Weights ride in the exponent: a p = sign(a)
// exp2(s k - (lse - log |a|)). fp32: less log2 of the row's scale over CS_XREF too, the scale of rows near 1
// (a small correction, so the statistics keep their low bits).
enum { CS_LSE2 = 0, CS_KX = 1, CS_LAB = 2, CS_LQ = 3 };
constexpr int CS_XREF = 13;
__host__ __device__ inline int64_t cs_stat(int64_t n, int a) { return (n >> 5) * 128 + a * 32 + (n & 31); }

// fp32: an item's scale 2^e, per 32 items three arrays of 32 words: f = 2^(-e - 1), the factor of its scores;
// -log2 f; and 2^15 f, the factor of its exponentials in the row pass's second product. e = 3 + 8 i brings the
// item's largest entry into [2^6, 2^14) (i = 1: entries from 2^-5 to 2^3): neighbours mostly share it, and what they
// share costs no work per score (forward of 4096 x 20k x 64: 98 us with one scale, 106 with items over 16 binades;
// 8192 x 100k x 128: 1.03 ms and 1.02). An item with an entry that is not finite has f = 2^90 and infinity (NaN, if one
// of them is) for -log2 f, and +-2^14 for its infinite entries, zeros for the others. e lies between -113 (2^15 for
// the largest number) and 99 (2^-27 for the smallest normal one). The row pass's exponentials are 2^(s - m - e0), m
// the running maximum of s + log2 f, e0 a group's -log2 f where its items share it, up to 28 (most exponentials are at
// most 1 then, and round as little as can be), else the common window's 12 or, with an item of 2^115 and more, zero: a
// row's likeliest item stays within 2^-124 and 2^100.
enum { CS_WF = 0, CS_WE = 1, CS_WP = 2 };
constexpr int CS_WE_MIN = -113, CS_WE_MAX = 99;
constexpr float CS_WE_REF = 12.f, CS_WE_FAR = 28.f, CS_WE_BIG = -100.f;
__host__ __device__ inline int64_t cs_wstat(int64_t v, int a) { return (v >> 5) * 96 + a * 32 + (v & 31); }

struct CsPass {
  const char* R;          // resident rows [nR][D] (plane stride r_plane bytes)
  const char* T;          // streamed rows [nT][D]
  int64_t nR, nT, t_last; // valid rows; the last streamed row that may be read
  int64_t r_plane, t_plane;
  int64_t r_ld, t_ld;     // bytes per row
  int r_ch, t_ch;         // 16-byte chunks a row holds (the rest of the kernel's width reads as zero)
  const char* zero;       // 16 zero bytes
  int64_t tiles, per;     // streamed tiles, tiles per split
  int full, nsplit, nrb;  // the first `full` resident blocks are not split, the other nrb are
  const CsScal* scal;
  float scale, kbase;     // c, c log2 e
  const float* kr;        // fp32: factors of the resident rows (row pass: 2^-e of x's rows, column pass: w's statistics)
  const int32_t* lab;     // row pass: label of each resident row (< 0: none)
  const float* stat;      // statistics of the streamed rows (column pass; fp32's row pass)
  int64_t pR;             // rows of the partials: those of the split blocks (full = 0: all, split or not)
  float *m, *O;           // partials m, l [pR][split], O [split][pR][D]
  double* l;
  // column pass: the gradient of the unsplit blocks
  void* out;
  int64_t ld;             // its row length
  int out_bf16;
  const float* gscale;
  const float* dx_unit;   // the forward's unit gradient of x, n_dx values: workgroups past the blocks scale it
  int64_t n_dx;           // (one launch less than a kernel of its own)
  void* dx;
};

template <int NP>
__device__ __forceinline__ f32x4 cs_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (NP == 1) return mfma16_bf16(a, b, c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(cs_h8, a), __builtin_bit_cast(cs_h8, b), c, 0, 0, 0);
}

// LDS image of a tile: bands of 8 rows, each D / 32 subtiles of 8 rows x 64 bytes; the four 16-B chunks of
// a subtile row are permuted by XOR with cs_swz(band). The row reads (16 rows of two or four bands, one
// chunk) and the transposed reads (16 rows, 32 bytes) then touch every bank evenly, and each kind needs
// one or two per-lane addresses, the rest being instruction offsets.
__device__ __forceinline__ int cs_swz(int band) { return ((((band) ^ (band >> 1)) & 1) << 1) | ((band >> 1) & 1); }

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

// the same from a uniform address plus 16 lane
__device__ __forceinline__ void cs_glds16u(const char* g, int lane, uint32_t dst) {
  const uint32_t m0v = __builtin_amdgcn_readfirstlane(dst);
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(16 * lane), "s"(g), "s"(m0v)
               : "memory");
}

// 2^m, an integer exponent (for ldexp) apart from a factor of one binade: an item that no row expects has
// an m far below the smallest number while its gradient is none of these
__device__ __forceinline__ int cs_exp2_split(float m, float& frac) {
  const float i = fmaxf(floorf(m), -1000.f);
  frac = __builtin_amdgcn_exp2f(fmaxf(m, -1000.f) - i);
  return (int)i;
}

// 2^d of a difference of two maxima, d <= 0. fp32's maxima are of scaled terms: 2^d may be below the smallest fp32 number
// where the sum it multiplies is far above one
template <int NP>
__device__ __forceinline__ double cs_exp2_d(float d) {
  if (NP == 1) return (double)__builtin_amdgcn_exp2f(d);
  const double h = (double)__builtin_amdgcn_exp2f(0.5f * d);
  return h * h;
}

// a pair of bf16, those that are not finite replaced by the largest number of their sign
__device__ __forceinline__ uint32_t cs_finite_bf16(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w = (w & 0xffff8000u) | 0x7f7fu;
  if ((w & 0x7f800000u) == 0x7f800000u) w = (w & 0x8000ffffu) | 0x7f7f0000u;
  return w;
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

// Shape of a pass: UB 16-row subtiles of resident rows per wave, NW waves, tiles of KT streamed rows taken
// in groups of 32 SG rows, NB tiles in LDS (the copies run NB - 1 tiles ahead), WG workgroups per CU.
// O, the resident rows and a group's scores fill the registers. Groups of 64 rows form half as many sums
// and maxima as groups of 32 (8192 x 100k x 128 fp32, forward: 0.97 against 1.19 ms). Three waves a SIMD
// where they fit: at 64 columns (8192 x 100k fp32, forward and backward: 0.59 and 0.56 ms against 0.60 and 0.59
// with two), and for the bf16 column pass, without a running maximum, at groups of 32 (16384 x 1M x 128: 6.2
// against 6.8 ms; 4096 x 60k x 256: 260 against 315 us). At 256 columns a wave holds 16 rows: 32 leave one wave a
// SIMD (4096 x 60k x 256 fp32: 697 and 727 against 641 and 632 us).
struct CsCfg {
  int UB, NW, KT, NB, SG, WG;
};
constexpr CsCfg cs_cfg(int D, int NP, int MODE) {
  if (D == 64) return {2, 4, 64, 3, 2, 3};
  if (NP == 1 && MODE == CS_COL) return D == 128 ? CsCfg{2, 4, 64, 2, 1, 3} : CsCfg{1, 4, 32, 3, 1, 3};
  if (D == 128) return {2, 8, 64, NP == 2 ? 4 : 8, 2, 1};
  return {1, 8, 64, NP == 2 ? 2 : 4, 2, 1};
}
constexpr int cs_block_rows(int D, int NP, int MODE) {
  return 16 * cs_cfg(D, NP, MODE).UB * cs_cfg(D, NP, MODE).NW;
}

// waves per SIMD its registers are budgeted for
constexpr int cs_lb(int D, int NP, int MODE) { return cs_cfg(D, NP, MODE).WG * cs_cfg(D, NP, MODE).NW / 4; }

// Steps that a product's LDS reads run ahead of its matrix instructions: fp32 has three instructions a
// step to hide them behind and no registers for more than one, bf16 one
enum { CS_S, CS_P };
constexpr int cs_ahead(int NP, int which) { return NP == 2 ? 1 : which == CS_S ? 2 : 4; }

template <int N>
__device__ __forceinline__ void cs_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// dx = c g / Z times the forward's unit gradient, `threads` values of 4 a workgroup
__device__ __forceinline__ void cs_dx(int64_t blk, int threads, const float* __restrict__ u, int64_t n, float scale,
                                      const CsScal* scal, const float* gscale, void* __restrict__ out, int bf16) {
  const float f = scale * scal->inv_z * (gscale ? *gscale : 1.f);
  const int64_t i = (blk * threads + threadIdx.x) * 4;
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

template <int D, int NP, int MODE>
__global__ __launch_bounds__(64 * cs_cfg(D, NP, MODE).NW, cs_lb(D, NP, MODE)) void cs_pass_kernel(CsPass p) {
  constexpr int UB = cs_cfg(D, NP, MODE).UB, NW = cs_cfg(D, NP, MODE).NW, KT = cs_cfg(D, NP, MODE).KT;
  constexpr int NB = cs_cfg(D, NP, MODE).NB;
  constexpr int ROWB = 2 * D, PLANE = KT * ROWB, IMG = NP * PLANE, NDT = D / 16, NC = D / 32;
  constexpr int SROW = MODE == CS_COL ? 16 : NP == 2 ? 12 : 0;  // bytes of statistics per streamed row
  constexpr int STAT = KT * SROW, BUF = IMG + STAT;
  constexpr bool RUNMAX = MODE != CS_COL || NP == 2;
  __shared__ __attribute__((aligned(1024))) char smem[NB * BUF];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, i16 = lane & 15;
  const int grid = p.full + p.nrb * p.nsplit;
  if (MODE == CS_COL && (int)blockIdx.x >= grid) {
    cs_dx(blockIdx.x - grid, 64 * NW, p.dx_unit, p.n_dx, p.scale, p.scal, p.gscale, p.dx, p.out_bf16);
    return;
  }
  const bool whole = (int)blockIdx.x < p.full;
  const int id = whole ? cs_xcd(blockIdx.x, p.full) : cs_xcd(blockIdx.x - p.full, grid - p.full);
  const int split = whole ? 0 : id / p.nrb;
  const int64_t r0 = (int64_t)(whole ? id : p.full + id % p.nrb) * cs_block_rows(D, NP, MODE) + wave * (16 * UB);
  const int64_t per = whole ? p.tiles : p.per;
  const int64_t tb0 = split * per, tb1 = tb0 + per < p.tiles ? tb0 + per : p.tiles;
  const uint32_t lds0 = (uint32_t) reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem);

  constexpr int SG = cs_cfg(D, NP, MODE).SG, GROUPS = KT / (32 * SG);
  constexpr int CPT = PLANE / (NW * 1024);       // 16-B copies per thread and plane of a tile
  constexpr int AHEAD = NB - 1;                  // tiles copied ahead
  static_assert(CPT >= 1 && KT % (32 * SG) == 0 && AHEAD >= 1, "tile shape");
  // this thread's copies of the next tile; a chunk past the rows' width comes from the zeros
  const char* src[CPT];
  int32_t src_step[CPT];
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    const int at = i * NW * 64 + tid, band = at / D;  // 16-B chunk of the image
    const int row = band * 8 + (at % 32) / 4, ch = (at % D) / 32 * 4 + ((at & 3) ^ cs_swz(band & 3));
    const bool in = NP == 2 || ch < p.t_ch;  // fp32's image has the whole width
    src[i] = in ? p.T + (tb0 * KT + row) * p.t_ld + ch * 16 : p.zero;
    src_step[i] = in ? (int32_t)(KT * p.t_ld) : 0;
  }
  auto copy = [&](int64_t t, int buf) __attribute__((always_inline)) {
    const int64_t over = t * KT + KT - 1 - p.t_last;  // rows of the tile past the last one repeat it
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const char* q = src[i];
      if (over > 0) {
        const int row = (i * NW * 64 + tid) / D * 8 + ((i * NW * 64 + tid) % 32) / 4;
        const int64_t back = row + over - (KT - 1);
        if (back > 0 && src_step[i]) q -= back * p.t_ld;
      }
#pragma unroll
      for (int pl = 0; pl < NP; ++pl)
        cs_glds16(q + pl * p.t_plane, lds0 + buf * BUF + pl * PLANE + i * NW * 1024 + wave * 1024);
      src[i] += src_step[i];
    }
    if constexpr (SROW > 0)
      if (wave == 0 && lane < STAT / 16) {
        if constexpr (NP == 2) cs_glds16u((const char*)p.stat + t * STAT, lane, lds0 + buf * BUF + IMG);
        else cs_glds16((const char*)p.stat + t * STAT + lane * 16, lds0 + buf * BUF + IMG);
      }
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (tb0 + i < tb1) copy(tb0 + i, i);

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
        xq[ub][c][pl] = *reinterpret_cast<const u32x4*>(
            4 * c + g < p.r_ch ? p.R + pl * p.r_plane + q * p.r_ld + (4 * c + g) * 16 : p.zero);
    // bf16: an infinite item becomes the largest finite one. Its probabilities are zero (or NaN, by the row's lse)
    // either way, but the zeros of a row that takes no part stay zeros.
    if constexpr (MODE == CS_COL && NP == 1)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) xq[ub][c][0][j] = cs_finite_bf16(xq[ub][c][0][j]);
    if constexpr (MODE != CS_COL) {
      // FLT_MIN: a masked item's -inf must stay -inf after the product
      kq[ub] = NP == 2 ? fminf(fmaxf(2.f * p.kbase * p.kr[q], FLT_MIN), FLT_MAX) : p.kbase;
      lab[ub] = p.lab[q];
    } else if constexpr (NP == 2) {
      kq[ub] = p.kr[cs_wstat(q, CS_WF)];
    }
  }
  // the resident rows are waited for here: a wait inside the loop would also wait for every copy in flight
#pragma unroll
  for (int ub = 0; ub < UB; ++ub) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int pl = 0; pl < NP; ++pl) asm volatile("" : "+v"(xq[ub][c][pl]));
    if constexpr (MODE != CS_COL) asm volatile("" : "+v"(kq[ub]), "+v"(lab[ub]));
    else if constexpr (NP == 2) asm volatile("" : "+v"(kq[ub]));
  }
  // fp32's column pass: the wave's items share a scale, or have one each (kq)
  bool same = true;
  float f0 = 1.f;
  if constexpr (MODE == CS_COL && NP == 2) {
    f0 = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, kq[0])));
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) same &= !__any(kq[ub] != f0);
  }
  const float kw = p.kbase;
  const float ps = NP == 2 && MODE == CS_COL ? CS_PS : 0.f;  // (the row pass's items bring it)
  const bool flip = MODE == CS_COL && p.scal->neg;

  // row reads: A row i16 of subtile kb = row 8 (i16 / 4) + 4 kb + i16 % 4 of 32, chunk 4 c + g
  auto row_at = [&](int ln) __attribute__((always_inline)) {
    const int g = ln >> 4, i16 = ln & 15;
    return lds0 + (i16 >> 2) * (8 * ROWB) + (i16 & 3) * 64 + (g ^ cs_swz(i16 >> 2)) * 16;
  };
  // transposed reads: row 8 g + 4 h + i16 / 4 of 32, columns 16 dt + 4 (i16 % 4) .., by o = dt % 2
  auto col_at = [&](int ln, int o) __attribute__((always_inline)) {
    const int g = ln >> 4, i16 = ln & 15;
    return lds0 + g * (8 * ROWB) + (i16 >> 2) * 64 + ((2 * o + ((i16 & 3) >> 1)) ^ cs_swz(g)) * 16 + 8 * (i16 & 1);
  };

  f32x4 O[MODE == CS_STATS ? 1 : NDT][UB];
#pragma unroll
  for (int dt = 0; dt < (MODE == CS_STATS ? 1 : NDT); ++dt)
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) O[dt][ub] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m[UB];   // the maximum of log2 terms, less ps
  double l[UB];  // this lane's sum (a million items' terms, one group's sum at a time)
#pragma unroll
  for (int ub = 0; ub < UB; ++ub) {
    m[ub] = CS_MIN;
    l[ub] = 0.;
  }
  struct Scores {
    f32x4 v[2 * SG][UB];  // [2 sub + kb][ub]: streamed row 32 sub + 8 g + 4 kb + r, resident row 16 ub + i16
  };
  struct Probs {
    u32x4 w[SG][UB][NP];  // the second product's B operand: k = 8 g + j of sub, j < 4 from kb = 0
  };

  // S of the group's streamed rows at LDS byte bo, one step = 32 columns of 32 rows
  auto scores = [&](int ln, uint32_t bo, Scores& s) __attribute__((always_inline)) {
    uint32_t at = row_at(ln) + bo;
    asm("" : "+v"(at));  // the offsets below stay in the instructions
    constexpr int NST = SG * NC, AH = cs_ahead(NP, CS_S);
    u32x4 a[AH + 1][2][NP];
    auto read = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int pl = 0; pl < NP; ++pl)
          a[j % (AH + 1)][kb][pl] = cs_lds<u32x4>(at + (j / NC) * (32 * ROWB) + (j % NC) * 512 + kb * 256 + pl * PLANE);
    };
#pragma unroll
    for (int j = 0; j < AH && j < NST; ++j) read(j);
#pragma unroll
    for (int j = 0; j < NST; ++j) {
      const int c = j % NC;
      if (j + AH < NST) read(j + AH);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
          f32x4& o = s.v[2 * (j / NC) + kb][ub];
          f32x4 z = {0.f, 0.f, 0.f, 0.f};
          if (c > 0) z = o;
          if constexpr (NP == 2) {
            z = cs_mfma<NP>(a[j % (AH + 1)][kb][1], xq[ub][c][0], z);
            z = cs_mfma<NP>(a[j % (AH + 1)][kb][0], xq[ub][c][1], z);
          }
          o = cs_mfma<NP>(a[j % (AH + 1)][kb][0], xq[ub][c][0], z);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // O += P times the group's rows. fp32 operands: the group's sum in fresh accumulators, then one fp32
  // multiply-add that also brings O to the scale P was formed at.
  auto product = [&](int ln, uint32_t bo, const Probs& pb, const float (&al)[UB]) __attribute__((always_inline)) {
    uint32_t at[2] = {col_at(ln, 0) + bo, NP == 2 ? (col_at(ln, 0) + bo) ^ 32 : col_at(ln, 1) + bo};  // (o is bit 5)
    asm("" : "+v"(at[0]), "+v"(at[1]));
    constexpr int NST = SG * NDT, AH = cs_ahead(NP, CS_P);
    u32x4 a[AH + 1][NP];
    f32x4 f[UB];
    auto read = [&](int j) __attribute__((always_inline)) {
      const int dt = j / SG;
#pragma unroll
      for (int pl = 0; pl < NP; ++pl)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const ib_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) ib_s16x4*)(uintptr_t)(at[dt & 1] + (j % SG) * (32 * ROWB) +
                                                                       (dt >> 1) * 512 + h * 256 + pl * PLANE));
          const u32x2 w2 = __builtin_bit_cast(u32x2, v);
          a[j % (AH + 1)][pl][2 * h] = w2[0];
          a[j % (AH + 1)][pl][2 * h + 1] = w2[1];
        }
    };
#pragma unroll
    for (int j = 0; j < AH && j < NST; ++j) read(j);
#pragma unroll
    for (int j = 0; j < NST; ++j) {
      const int dt = j / SG, sub = j % SG;
      if (j + AH < NST) read(j + AH);
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) {
        if constexpr (NP == 2) {
          if (sub == 0) f[ub] = f32x4{0.f, 0.f, 0.f, 0.f};
          f[ub] = cs_mfma<NP>(a[j % (AH + 1)][1], pb.w[sub][ub][0], f[ub]);
          f[ub] = cs_mfma<NP>(a[j % (AH + 1)][0], pb.w[sub][ub][1], f[ub]);
          f[ub] = cs_mfma<NP>(a[j % (AH + 1)][0], pb.w[sub][ub][0], f[ub]);
          if (sub == SG - 1) O[dt][ub] = O[dt][ub] * al[ub] + f[ub];
        } else {
          O[dt][ub] = cs_mfma<NP>(a[j % (AH + 1)][0], pb.w[sub][ub][0], O[dt][ub]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // four probabilities of subtile k -> words of P (fp32's row pass: times the items' factors f, the products
  // part of the two roundings)
  auto pack = [&](Probs& pb, int k, int ub, f32x4 e, f32x4 f) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float a = e[2 * h], b = e[2 * h + 1];
      const int w = 2 * (k & 1) + h;
      if constexpr (NP == 1) pb.w[k >> 1][ub][0][w] = ib_pk(a, b);
      else if constexpr (MODE == CS_ROW) {
        const float fa = f[2 * h], fb = f[2 * h + 1];
        const cs_h2 hi = __builtin_bit_cast(cs_h2, __builtin_amdgcn_cvt_pkrtz(a * fa, b * fb));
        pb.w[k >> 1][ub][0][w] = __builtin_bit_cast(uint32_t, hi);
        pb.w[k >> 1][ub][1][w] =
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf(a, fa, -(float)hi[0]),
                                                                    __builtin_fmaf(b, fb, -(float)hi[1])));
      } else {
        const cs_h2 hi = __builtin_bit_cast(cs_h2, __builtin_amdgcn_cvt_pkrtz(a, b));
        pb.w[k >> 1][ub][0][w] = __builtin_bit_cast(uint32_t, hi);
        pb.w[k >> 1][ub][1][w] =
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a - (float)hi[0], b - (float)hi[1]));
      }
    }
  };
  // statistic a of subtile k's streamed rows, sg = a group's statistics plus 32 g
  auto stat_at = [&](uint32_t sg, int a, int k) __attribute__((always_inline)) {
    return sg + (k >> 1) * (32 * SROW) + a * 128 + (k & 1) * 16;
  };
  // f(k, ub, r, whether this element is its streamed row's label, x(k)[r])
  auto each_hit = [&](uint32_t sg, auto&& x, auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2 * SG; ++k) {
      const u32x4 lb = cs_lds<u32x4>(stat_at(sg, CS_LAB, k));
      const f32x4 xk = x(k);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int32_t at = ((int32_t)lb[r] >> 1) - ((int32_t)r0 + i16);
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) f(k, ub, r, at == 16 * ub, xk[r]);
      }
    }
  };
  // Before a group's exponentials (its first streamed row is n0): the label's term leaves them and the
  // running maximum is raised (up, al: what that multiplies O and l by). Both are rare, and what they
  // change is small, so the common path has no branch between its matrix and vector instructions.
  auto prepare = [&](int64_t n0, int ln, uint32_t st, uint32_t sg, Scores& s, float (&al)[UB], float (&kg)[UB],
                     float& e0, bool& up, bool& hit) __attribute__((always_inline)) {
    up = hit = false;
    bool one = true;
    float ew = 0.f;  // -log2 f of the group's items, where they share it
    if constexpr (MODE == CS_COL) {
      if constexpr (NP == 2) {
        // log2 p = s k_n f_v - lse2_n (s k_n first: that is finite in a row that takes no part, which has k_n = 1)
        if (same) {
#pragma unroll
          for (int k = 0; k < 2 * SG; ++k) {
            const f32x4 ls = cs_lds<f32x4>(stat_at(sg, CS_LSE2, k)), kn = cs_lds<f32x4>(stat_at(sg, CS_KX, k)) * f0;
#pragma unroll
            for (int ub = 0; ub < UB; ++ub)
#pragma unroll
              for (int r = 0; r < 4; ++r) s.v[k][ub][r] = __builtin_fmaf(s.v[k][ub][r], kn[r], -ls[r]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 2 * SG; ++k) {
            const f32x4 ls = cs_lds<f32x4>(stat_at(sg, CS_LSE2, k)), kn = cs_lds<f32x4>(stat_at(sg, CS_KX, k));
#pragma unroll
            for (int ub = 0; ub < UB; ++ub)
#pragma unroll
              for (int r = 0; r < 4; ++r) s.v[k][ub][r] = __builtin_fmaf(s.v[k][ub][r] * kn[r], kq[ub], -ls[r]);
          }
        }
      }
      const int ll = ln & (32 * SG - 1);
      const int32_t lb = cs_lds<int32_t>(st + (ll >> 5) * 512 + CS_LAB * 128 + (ll & 31) * 4) >> 1;
      hit = __any((uint32_t)(lb - (int32_t)r0) < (uint32_t)(16 * UB));
      // fp32: the label's element is to become |a| q (its sign follows in `patch`); the scores are log2 p here
      if (NP == 2 && hit) {
        asm volatile("");  // keeps the rare path a branch
        each_hit(sg, [&](int k) __attribute__((always_inline)) { return cs_lds<f32x4>(stat_at(sg, CS_LQ, k)); },
                 [&](int k, int ub, int r, bool is, float x) __attribute__((always_inline)) {
                   s.v[k][ub][r] = is ? x : s.v[k][ub][r];
                 });
      }
    } else {
      if constexpr (NP == 2) {
        // the items' scales: one for the group, or one each (then in the scores, the group's being 1)
        const int ll = ln & (32 * SG - 1);
        const float we = cs_lds<float>(st + (ll >> 5) * (32 * SROW) + CS_WE * 128 + (ll & 31) * 4);
        e0 = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, we)));
        one = e0 < INFINITY && !__any(!(we == e0));
        if (!one) {
          asm volatile("");  // keeps the rare path a branch
          e0 = __any(we < CS_WE_BIG) ? 0.f : CS_WE_REF;
#pragma unroll
          for (int k = 0; k < 2 * SG; ++k) {
            const f32x4 f = cs_lds<f32x4>(stat_at(sg, CS_WF, k)), w = cs_lds<f32x4>(stat_at(sg, CS_WE, k));
#pragma unroll
            for (int ub = 0; ub < UB; ++ub)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                // an item that is not finite: a score of -infinity leaves the sum, any other is NaN
                const float x = s.v[k][ub][r] * f[r], y = x * w[r];
                s.v[k][ub][r] = w[r] < INFINITY ? x : y < 0.f ? y : NAN;
              }
          }
        }
        const float f0 = one ? __builtin_bit_cast(float, (127 - (int)e0) << 23) : 1.f;
        ew = e0;
        if (one) e0 = fminf(e0, CS_WE_FAR);
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) kg[ub] = fminf(fmaxf(kq[ub] * f0, FLT_MIN), FLT_MAX);
      }
      bool mine = false;
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) mine |= (uint32_t)(lab[ub] - (int32_t)n0) < 32u * SG;
      if (__any(mine) || n0 + 32 * SG > p.nT) {
        const int32_t base = (int32_t)n0 + 8 * g, left = (int32_t)p.nT - base;
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
          const int32_t at = lab[ub] - base;
#pragma unroll
          for (int k = 0; k < 2 * SG; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int v = 32 * (k >> 1) + 4 * (k & 1) + r;
              s.v[k][ub][r] = v >= left || v == at ? -INFINITY : s.v[k][ub][r];
            }
        }
      }
    }
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) al[ub] = 1.f;
    if constexpr (RUNMAX) {
      float mx[UB];
      bool mine = false;
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) {
        float z = fmaxf(s.v[0][ub][0], s.v[0][ub][1]);
#pragma unroll
        for (int k = 0; k < 2 * SG; ++k)
#pragma unroll
          for (int r = k == 0 ? 2 : 0; r < 4; r += 2) z = fmaxf(fmaxf(s.v[k][ub][r], s.v[k][ub][r + 1]), z);
        mx[ub] = MODE == CS_COL ? z : NP == 1 ? z * kq[ub] : __builtin_fmaf(z, kg[ub], -ew);
      }
      if constexpr (MODE != CS_COL && NP == 2)  // the maximum is that of exp s times the item's factor
        if (!one) {
          asm volatile("");  // keeps the rare path a branch
#pragma unroll
          for (int ub = 0; ub < UB; ++ub) mx[ub] = -INFINITY;
#pragma unroll
          for (int k = 0; k < 2 * SG; ++k) {
            const f32x4 w = cs_lds<f32x4>(stat_at(sg, CS_WE, k));
#pragma unroll
            for (int ub = 0; ub < UB; ++ub)
#pragma unroll
              for (int r = 0; r < 4; ++r) mx[ub] = fmaxf(__builtin_fmaf(s.v[k][ub][r], kg[ub], -w[r]), mx[ub]);
          }
        }
#pragma unroll
      for (int ub = 0; ub < UB; ++ub) {
        mx[ub] -= ps;
        mine |= mx[ub] > m[ub];
      }
      up = __any(mine);
      if (up) {
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
          float x = fmaxf(mx[ub], __shfl_xor(mx[ub], 16, 64));
          x = fmaxf(x, __shfl_xor(x, 32, 64));
          if (MODE != CS_COL && NP == 2) x = ceilf(x);  // m + e0 is exact
          x = fmaxf(x, m[ub]);
          al[ub] = __builtin_amdgcn_exp2f(m[ub] - x);
          l[ub] *= cs_exp2_d<NP>(m[ub] - x);
          m[ub] = x;
        }
      }
    }
  };
  // The label's element of P is negative. bf16: it is set here to |a| q rounded, and `rest` leaves what that rounding
  // lost as a P of its own: the label's term is most of an item's gradient where it has one.
  auto patch = [&](uint32_t sg, Probs& pb, bool rest) __attribute__((always_inline)) {
    if constexpr (NP == 2) {
      each_hit(sg, [](int) { return f32x4{}; }, [&](int k, int ub, int r, bool is, float) __attribute__((always_inline)) {
        const uint32_t sign = is ? (r & 1 ? 0x80000000u : 0x8000u) : 0u;
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) pb.w[k >> 1][ub][pl][2 * (k & 1) + (r >> 1)] ^= sign;
      });
    } else {
      each_hit(sg,
               [&](int k) __attribute__((always_inline)) {
                 f32x4 v = cs_lds<f32x4>(stat_at(sg, CS_LQ, k));
#pragma unroll
                 for (int r = 0; r < 4; ++r) {
                   const float q = __builtin_amdgcn_exp2f(v[r]), h = (float)(__bf16)q;
                   v[r] = rest ? h - q : -h;
                 }
                 return v;
               },
               [&](int k, int ub, int r, bool is, float x) __attribute__((always_inline)) {
                 const int i = 2 * (k & 1) + (r >> 1);
                 const uint32_t keep = r & 1 ? 0xffffu : 0xffff0000u, bits = ib_pk(r & 1 ? 0.f : x, r & 1 ? x : 0.f);
                 const uint32_t w = pb.w[k >> 1][ub][0][i];
                 pb.w[k >> 1][ub][0][i] = is ? (w & keep) | (bits & ~keep) : w;
               });
    }
  };
  // rows of negative weight
  auto negate = [&](uint32_t sg, Probs& pb) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2 * SG; ++k) {
      const u32x4 lb = cs_lds<u32x4>(stat_at(sg, CS_LAB, k));
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int ub = 0; ub < UB; ++ub)
#pragma unroll
          for (int pl = 0; pl < NP; ++pl)
            pb.w[k >> 1][ub][pl][2 * (k & 1) + h] ^= ((lb[2 * h] & 1) << 15) | ((lb[2 * h + 1] & 1) << 31);
    }
  };
  // exponentials of part i = (subtile k, ub) of 2 SG UB
  auto exponentials = [&](int i, uint32_t sg, const Scores& s, Probs& pb, const float (&kg)[UB], const float (&mg)[UB],
                          float p0, float (&sum)[UB]) __attribute__((always_inline)) {
    const int k = i / UB, ub = i % UB;
    f32x4 ls, e, f = {};
    if constexpr (MODE == CS_COL && NP == 1) ls = cs_lds<f32x4>(stat_at(sg, CS_LSE2, k));
    if constexpr (MODE == CS_ROW && NP == 2) f = cs_lds<f32x4>(stat_at(sg, CS_WP, k)) * p0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = s.v[k][ub][r];
      if constexpr (MODE != CS_COL)
        e[r] = __builtin_amdgcn_exp2f(NP == 2 ? __builtin_fmaf(x, kg[ub], -mg[ub]) : __builtin_fmaf(x, kq[ub], -m[ub]));
      else if constexpr (NP == 2) e[r] = __builtin_amdgcn_exp2f(x - m[ub]);
      else e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, kw, -ls[r]));
    }
    if constexpr (MODE != CS_COL) sum[ub] += (e[0] + e[1]) + (e[2] + e[3]);
    if constexpr (MODE != CS_STATS) pack(pb, k, ub, e, f);
  };
  // O and l follow a raised maximum (bf16; with fp32 operands the product does it for O)
  auto rescale = [&](bool up, const float (&al)[UB]) __attribute__((always_inline)) {
    if constexpr (NP == 1 && MODE == CS_ROW)
      if (up)
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int ub = 0; ub < UB; ++ub) O[dt][ub] *= al[ub];
  };
  // The ring: at tile t's barrier its copies have landed and no wave reads tile t - 1 any more; the copy
  // that follows fills tile t - 1's buffer.
  const bool active = r0 < p.nR;  // a wave without rows only copies
  int buf = 0;
  for (int64_t t = tb0; t < tb1; ++t) {
    if (t + AHEAD > tb1) cs_wait<0>();
    else if (SROW > 0 && wave == 0) cs_wait<(AHEAD - 1) * (CPT * NP + 1)>();
    else cs_wait<(AHEAD - 1) * CPT * NP>();
    __syncthreads();
    if (t + AHEAD < tb1) copy(t + AHEAD, buf == 0 ? NB - 1 : buf - 1);
    if (active)
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        const int64_t n0 = t * KT + 32 * SG * gr;
        const uint32_t bo = buf * BUF + 32 * SG * gr * ROWB, st = lds0 + buf * BUF + IMG + 32 * SG * gr * SROW;
        int ln = lane;
        // fp32 has no registers to spare: what follows from the lane is formed here again, not held in registers (a
        // reload from scratch would also wait for the copies in flight), the statistics' offsets stay in the instructions
        if constexpr (NP == 2) asm volatile("" : "+v"(ln));
        uint32_t sg = st + 32 * (ln >> 4);
        if constexpr (NP == 2) asm("" : "+v"(sg));
        float al[UB], kg[UB], mg[UB], sum[UB] = {}, e0 = 0.f;
        bool up, hit;
        Scores s;
        Probs pb;
        scores(ln, bo, s);
        prepare(n0, ln, st, sg, s, al, kg, e0, up, hit);
        const float p0 = __builtin_bit_cast(float, (127 + (int)e0) << 23);
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) mg[ub] = m[ub] + e0;
        rescale(up, al);
#pragma unroll
        for (int i = 0; i < 2 * SG * UB; ++i) exponentials(i, sg, s, pb, kg, mg, p0, sum);
        if constexpr (MODE != CS_COL)
#pragma unroll
          for (int ub = 0; ub < UB; ++ub) l[ub] += NP == 2 ? (double)sum[ub] * (double)p0 : (double)sum[ub];
        if constexpr (MODE == CS_COL) {
          if (hit) {
            asm volatile("");  // keeps the rare path a branch
            patch(sg, pb, false);
          }
          if (flip) negate(sg, pb);
        }
        if constexpr (MODE != CS_STATS) product(ln, bo, pb, al);
        if constexpr (MODE == CS_COL && NP == 1)
          if (hit) {
            asm volatile("");  // keeps the rare path a branch
            pb = Probs{};
            patch(sg, pb, true);
            if (flip) negate(sg, pb);
            product(ln, bo, pb, al);
          }
      }
    buf = buf + 1 == NB ? 0 : buf + 1;
  }

#pragma unroll
  for (int ub = 0; ub < UB; ++ub) {
    const int64_t q = r0 + 16 * ub + i16;
    double sum = l[ub];
    if constexpr (MODE != CS_COL && NP == 1) {
      float f = (float)sum;
      f += __shfl_xor(f, 16, 64);
      f += __shfl_xor(f, 32, 64);
      sum = f;
    } else if constexpr (MODE != CS_COL) {  // may pass fp32's range
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
    }
    if (q >= p.nR) continue;
    if (MODE == CS_COL && whole) {
      // dw = O 2^m (x's scales are in the exponents), times c g / Z
      float f = p.scale * p.scal->inv_z * (p.gscale ? *p.gscale : 1.f);
      int ex = 0;
      if constexpr (NP == 2) {
        float frac;
        ex = cs_exp2_split(m[ub], frac) - CS_XREF;
        f *= frac;
      }
#pragma unroll
      for (int dt = 0; dt < (MODE == CS_STATS ? 1 : NDT); ++dt) {
        f32x4 v = O[dt][ub] * f;
        if constexpr (NP == 2)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], ex);
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
    const int64_t qp = q - (int64_t)p.full * cs_block_rows(D, NP, MODE);
    if (g == 0) {
      if constexpr (RUNMAX) p.m[qp * p.nsplit + split] = m[ub];
      if constexpr (MODE != CS_COL) p.l[qp * p.nsplit + split] = sum;
    }
    if constexpr (MODE != CS_STATS)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(p.O + (split * p.pR + qp) * D + 16 * dt + 4 * g) = O[dt][ub];
  }
}

// ---- the loss alone, few fp32 rows -----------------------------------------------------------------
// Up to 64 rows (256-wide: 32) against the catalogue: its bytes are the bound, so w is read once, as it lies (an image
// would read it twice and write it; so do the widths whose rows do not start on 16 bytes, for whose loads this kernel
// has no form), straight into the A operand of the fp32 matrix instruction (exact
// products; 16 items x 4 columns x 16 rows each), one step of 16 items ahead. A workgroup's four waves
// share a range of items; their maxima and sums join in LDS.
struct CsFew {
  const float *x, *w;
  const int64_t* labels;
  int64_t N, V, D, ignore;
  int64_t steps;  // of 64 items, dealt to the workgroups in turn
  float kbase;
  int32_t* lab;
  float* m;
  double* l;
  unsigned int* done;
};
template <int DP, int Q>
__global__ __launch_bounds__(256) void cs_few_kernel(CsFew p) {
  constexpr int NC = DP / 16;
  __shared__ float sh[2][4][16 * Q];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, i16 = lane & 15;
  // columns 16 c + 4 g .. of a row (D % 4 == 0): element j is the k = g operand of product (c, j)
  auto load = [&](const float* row, f32x4 (&v)[NC]) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = 16 * c + 4 * g;
      v[c] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (d < p.D) v[c] = *reinterpret_cast<const f32x4*>(row + d);
    }
  };
  if (blockIdx.x == 0) ticket_zero(p.done, threadIdx.x, 256);
  f32x4 xq[Q][NC];
  int32_t lab[Q];
  float m[Q], l[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int64_t n = 16 * q + i16 < p.N ? 16 * q + i16 : p.N - 1;
    load(p.x + n * p.D, xq[q]);
    const int64_t y = p.labels[n];
    lab[q] = y == p.ignore ? -1 : (y >= 0 && y < p.V) ? (int32_t)y : -2;
    if (blockIdx.x == 0 && wave == 0 && g == 0 && 16 * q + i16 < p.N) p.lab[n] = lab[q];
    if (lab[q] < 0) {  // an ignored row's finite entries only
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) xq[q][c][j] = fabsf(xq[q][c][j]) <= FLT_MAX ? xq[q][c][j] : 0.f;
    }
    m[q] = CS_MIN;
    l[q] = 0.f;
  }
  auto item = [&](int64_t step) __attribute__((always_inline)) {
    const int64_t v = step * 64 + wave * 16 + i16;
    return p.w + (v < p.V ? v : p.V - 1) * p.D;
  };
  f32x4 a[2][NC];
  auto step = [&](int64_t t, f32x4 (&now)[NC], f32x4 (&next)[NC]) __attribute__((always_inline)) {
    load(item(t + gridDim.x < p.steps ? t + gridDim.x : t), next);
    const int32_t v0 = (int32_t)(t * 64 + wave * 16 + 4 * g);  // accumulator element r is item v0 + r
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_16x16x4f32(now[c][j], xq[q][c][j], s, 0, 0, 0);
      s *= p.kbase;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (v0 + r >= p.V || v0 + r == lab[q]) s[r] = -INFINITY;
      const float x = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), m[q]);  // per lane: lanes join at the end
      float e = l[q] * __builtin_amdgcn_exp2f(m[q] - x);
#pragma unroll
      for (int r = 0; r < 4; ++r) e += __builtin_amdgcn_exp2f(s[r] - x);
      l[q] = e;
      m[q] = x;
    }
  };
  const int64_t G = gridDim.x;
  int64_t t = blockIdx.x;
  load(item(t), a[0]);
  for (; t + G < p.steps; t += 2 * G) {
    step(t, a[0], a[1]);
    step(t + G, a[1], a[0]);
  }
  if (t < p.steps) step(t, a[0], a[1]);
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    float x = fmaxf(m[q], __shfl_xor(m[q], 16, 64));
    x = fmaxf(x, __shfl_xor(x, 32, 64));
    float e = l[q] * __builtin_amdgcn_exp2f(m[q] - x);
    e += __shfl_xor(e, 16, 64);
    e += __shfl_xor(e, 32, 64);
    if (g == 0) {
      sh[0][wave][16 * q + i16] = x;
      sh[1][wave][16 * q + i16] = e;
    }
  }
  __syncthreads();
  const int n = threadIdx.x;
  if (n < 16 * Q && n < p.N) {
    float x = CS_MIN, e = 0.f;
    for (int k = 0; k < 4; ++k) x = fmaxf(x, sh[0][k][n]);
    for (int k = 0; k < 4; ++k) e += sh[1][k][n] * __builtin_amdgcn_exp2f(sh[0][k][n] - x);
    p.m[n * gridDim.x + blockIdx.x] = x;
    p.l[n * gridDim.x + blockIdx.x] = e;
  }
}

// ---- operand images ------------------------------------------------------------------------------
__device__ __forceinline__ float cs_finite_abs(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.f;
}
// the power of two that brings a into [2^13, 2^14)
__device__ __forceinline__ int cs_exp(float a) {
  if (!(a > 0.f)) return 0;
  int e;
  (void)frexpf(a, &e);  // a in [2^(e-1), 2^e)
  const int k = 14 - e;
  return k > 126 ? 126 : k;  // at least -114; both powers are normal numbers
}

struct CsImage {
  const void *x, *w;
  char *ximg, *wimg;       // wimg null: w is read as it is
  int64_t N, Npad, V, Vpad, D;
  int64_t xplane, wplane;
  int64_t ignore;
  const int64_t* labels;
  int32_t* lab;
  float *kx, *wstat;
  CsScal* scal;
  unsigned int* done;
  int xblocks;
};

// x [N, D] and w [V, D] into padded 16-bit rows: two fp16 planes of the scaled values (fp32), with w's
// statistics (up to a whole tile), or a copy (bf16). A row of x that takes no part keeps its finite entries only
// (its weight in the column pass is zero, and zero times infinity would not be). 4 columns per lane.
template <int DP, int NP>
__global__ __launch_bounds__(256) void cs_image_kernel(CsImage p) {
  constexpr int LPR = DP / 4, RPB = 256 / LPR;  // lanes per row, rows per workgroup
  const int c = (threadIdx.x % LPR) * 4, rr = threadIdx.x / LPR;
  const bool is_x = (int)blockIdx.x < p.xblocks;
  if (blockIdx.x == 0) {
    if (threadIdx.x < 4) p.scal->zero[threadIdx.x] = 0.f;
    ticket_zero(p.done, threadIdx.x, 256);
  }
  const int64_t blk = is_x ? blockIdx.x : blockIdx.x - p.xblocks;
  const int64_t nblk = is_x ? p.xblocks : gridDim.x - p.xblocks;
  const int64_t rows = is_x ? p.N : p.V, rows_pad = is_x ? p.Npad : NP == 2 ? p.Vpad : p.V;
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
      if (r < rows) {
        if (vec) {
          if (c < p.D) {
            const u32x2 q = *reinterpret_cast<const u32x2*>(s);
            h[0] = (uint16_t)q[0], h[1] = (uint16_t)(q[0] >> 16), h[2] = (uint16_t)q[1], h[3] = (uint16_t)(q[1] >> 16);
          }
        } else {
          for (int j = 0; j < 4; ++j)
            if (c + j < p.D) h[j] = s[j];
        }
        if (is_x && lb < 0)
          for (int j = 0; j < 4; ++j)
            if ((h[j] & 0x7f80) == 0x7f80) h[j] = 0;
      }
      *reinterpret_cast<u32x2*>(dst + r * (2 * DP) + 2 * c) =
          u32x2{h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16)};
    } else {
      const float* s = (const float*)src + (is_x || r < rows ? r : rows - 1) * p.D + c;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (!is_x || r < rows) {
        if (vec) {
          if (c < p.D) v = *reinterpret_cast<const f32x4*>(s);
        } else {
          for (int j = 0; j < 4; ++j)
            if (c + j < p.D) v[j] = s[j];
        }
      }
      if (is_x && lb < 0)
        for (int j = 0; j < 4; ++j) v[j] = fabsf(v[j]) <= FLT_MAX ? v[j] : 0.f;
      float a = fmaxf(fmaxf(cs_finite_abs(v[0]), cs_finite_abs(v[1])), fmaxf(cs_finite_abs(v[2]), cs_finite_abs(v[3])));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
      int e = cs_exp(a);
      if (is_x) {
        if (c == 0) p.kx[r] = ldexpf(1.f, -e);
      } else {
        e = !(a > 0.f) || e > CS_WE_MAX ? CS_WE_MAX : ((e - 3) & ~7) + 3;
        e = e < CS_WE_MIN ? CS_WE_MIN : e;
        int odd = 0;  // 1: an infinite entry, 2: a NaN
        for (int j = 0; j < 4; ++j) odd = isnan(v[j]) ? 2 : isinf(v[j]) && odd < 1 ? 1 : odd;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
          const int b = __shfl_xor(odd, o, 64);
          odd = odd > b ? odd : b;
        }
        if (odd) {
          e = 0;
          for (int j = 0; j < 4; ++j) v[j] = isinf(v[j]) ? copysignf(0x1p14f, v[j]) : 0.f;
        }
        if (c == 0) {
          p.wstat[cs_wstat(r, CS_WF)] = odd ? 0x1p90f : ldexpf(1.f, -e - 1);
          p.wstat[cs_wstat(r, CS_WE)] = odd == 2 ? NAN : odd ? INFINITY : (float)(e + 1);
          p.wstat[cs_wstat(r, CS_WP)] = ldexpf(1.f, 14 - e);
        }
        if (r >= rows) continue;  // past the last item: its statistics again, so that its group keeps one scale
      }
      const float sc = ldexpf(1.f, e);
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
  const float *m, *O;
  const double* l;
  const int32_t* lab;
  const float* weights;
  const float* kx;
  float scale, kbase;
  float *row, *lse, *dx, *stat;
  char* ximg;
  CsScal* scal;
  unsigned int* done;  // completion tickets (ticket_last), or null: the total is another kernel's
  int mean;
  float* loss;
};
__device__ __forceinline__ float cs_ld(const void* x, int bf16, int64_t i) {
  return bf16 ? (float)((const __bf16*)x)[i] : ((const float*)x)[i];
}

// the loss, 1 / Z and whether a weight is negative: one workgroup, fixed order. The row losses may come
// from other workgroups of the same grid.
__device__ __forceinline__ void cs_total(const CsRows& p) {
  __shared__ double sh[2][16];
  __shared__ int neg;
  const int threads = blockDim.x, waves = threads / 64;
  if (threadIdx.x == 0) neg = 0;
  __syncthreads();
  double s = 0., z = 0.;
  bool below = false;
  constexpr int U = 8;  // loads in flight
  for (int64_t n0 = threadIdx.x; n0 < p.N; n0 += U * threads) {
    float r[U], a[U];
    int32_t lab[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * threads, i = n < p.N ? n : p.N - 1;
      r[u] = __hip_atomic_load(p.row + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      a[u] = p.weights ? p.weights[i] : 1.f;
      lab[u] = n < p.N ? p.lab[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = lab[u] != -1;
      below |= in && a[u] < 0.f;
      s += in ? (double)a[u] * (double)r[u] : 0.;
      z += in ? (double)a[u] : 0.;
    }
  }
  if (below) neg = 1;
  s = wave_sum_d(s);
  z = wave_sum_d(z);
  if ((threadIdx.x & 63) == 0) {
    sh[0][threadIdx.x >> 6] = s;
    sh[1][threadIdx.x >> 6] = z;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = z = 0.;
    for (int i = 0; i < waves; ++i) {
      s += sh[0][i];
      z += sh[1][i];
    }
    const double inv = !p.mean ? 1. : z != 0. ? 1. / z : 0.;
    p.scal->inv_z = (float)inv;
    p.scal->neg = neg;
    *p.loss = (float)(s * inv);
  }
}
__global__ __launch_bounds__(1024) void cs_total_kernel(CsRows p) { cs_total(p); }

// Joins the splits of a row: NWV waves per row (1: four rows per workgroup), DP / 4 lanes per split, the
// splits dealt to the lane groups and their sums joined in a fixed order. Then the label's logit (64-bit
// sums), the row's loss, its statistics for the column pass and its unit gradient a q (O / l - w_y).
template <int DP, int NP, int NWV>
__device__ __forceinline__ void cs_row(const CsRows& p) {
  constexpr int LPR = DP / 4, GW = 64 / LPR, G = NWV * GW;
  __shared__ f32x4 sh[NWV][LPR];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = NWV == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  const bool first = NWV == 1 || wave == 0;
  if (n >= p.Npad) return;
  if (n >= p.N) {
    if (first && lane == 0 && p.stat) {
      p.stat[cs_stat(n, CS_LSE2)] = INFINITY;
      p.stat[cs_stat(n, CS_KX)] = 1.f;
      reinterpret_cast<int32_t*>(p.stat)[cs_stat(n, CS_LAB)] = -1;
      p.stat[cs_stat(n, CS_LQ)] = 0.f;
    }
    return;
  }
  const int32_t lb = p.lab[n];
  const float* ms = p.m + n * p.nsplit;
  const int c = (lane % LPR) * 4;
  const float a = p.weights ? p.weights[n] : 1.f;
  float xv[4], wv[4];  // this lane's columns of x and of the label's item, asked for before the joins
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = lb >= 0 && c + j < p.D && first;
    xv[j] = in ? cs_ld(p.x, p.bf16, n * p.D + c + j) : 0.f;
    wv[j] = in ? cs_ld(p.w, p.bf16, (int64_t)lb * p.D + c + j) : 0.f;
  }
  float M = CS_MIN;
#pragma unroll 4
  for (int s = lane; s < p.nsplit; s += 64) M = fmaxf(M, ms[s]);
  M = wave_max(M);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (p.dx && lb >= 0) {
    const int64_t step = p.N * DP;
    const float* os = p.O + n * DP + c;
#pragma unroll 4
    for (int s = (NWV == 1 ? 0 : wave * GW) + lane / LPR; s < p.nsplit; s += G)
      o += *reinterpret_cast<const f32x4*>(os + s * step) * __builtin_amdgcn_exp2f(ms[s] - M);
#pragma unroll
    for (int k = LPR; k < 64; k <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], k, 64);
    if constexpr (NWV > 1) {
      if (lane < LPR) sh[wave][lane] = o;
      __syncthreads();
      if (wave == 0)
        for (int k = 1; k < NWV; ++k) o += sh[k][lane % LPR];
    }
  }
  if (!first) return;
  double L = 0.;
#pragma unroll 4
  for (int s = lane; s < p.nsplit; s += 64)
    L += p.l[n * p.nsplit + s] * cs_exp2_d<NP>(ms[s] - M);
  L = wave_sum_d(L);
  // in log2 units: the other items' log sum and the label's logit. Logarithms of fp32 mantissas (error
  // below 2^-23), sums with the exponents in 64 bits: the 64-bit logarithm, on every row, took most of
  // this kernel's time.
  int le = 0;
  const double lm = L > 0. && L < INFINITY ? frexp(L, &le) : L;
  const double o2 = L == 0. ? -INFINITY : (double)M + le + (double)__builtin_amdgcn_logf((float)lm);
  double sy = 0.;
#pragma unroll
  for (int j = 0; j < 4; ++j) sy += (double)xv[j] * (double)wv[j];
#pragma unroll
  for (int k = LPR / 2; k > 0; k >>= 1) sy += __shfl_xor(sy, k, 64);
  sy *= (double)p.scale * CS_LOG2E;
  // every item, the label's too, below the running maximum's start: what they are to one another is lost
  const bool lost = lb >= 0 && L == 0. && p.V > 1 && !(sy > 0.5 * CS_MIN);
  const float t = lost ? NAN : (float)((o2 - sy) * CS_LN2);
  const float et = expf(-fabsf(t)), soft = log1pf(et);
  const float q = t > 0.f ? 1.f / (1.f + et) : et / (1.f + et);  // NaN stays NaN
  const double lse2 = lb >= 0 ? fmax(o2, sy) + (double)soft * CS_LOG2E : o2;
  if (lane == 0) {
    __hip_atomic_store(p.row + n, lb >= 0 ? soft + fmaxf(t, 0.f) : lb == -1 ? 0.f : NAN, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);  // the grid's last workgroup sums them
    if (p.lse) p.lse[n] = (float)(lse2 * CS_LN2);
  }
  if (lane == 0 && p.stat) {  // a column pass follows
    const bool live = lb >= 0;
    double ca = log2f(fabsf(a));
    if (NP == 2) ca += ilogbf(p.kx[n]) + CS_XREF;
    // NaN statistics of a labelled row reach every item's gradient, as the formula's do; infinite is the statistic of a
    // weight of zero alone
    double ls = lse2 == INFINITY ? NAN : lse2 - ca;
    if (a != 0.f && !isnan(ls)) ls = fmin(fmax(ls, -(double)FLT_MAX), (double)FLT_MAX);
    p.stat[cs_stat(n, CS_LSE2)] = live ? (float)ls : INFINITY;
    // (a row that takes no part: a factor whose product with any score is finite)
    p.stat[cs_stat(n, CS_KX)] = NP == 2 && live ? fminf(fmaxf(2.f * p.kbase * p.kx[n], FLT_MIN), FLT_MAX) : 1.f;
    reinterpret_cast<int32_t*>(p.stat)[cs_stat(n, CS_LAB)] = live ? 2 * lb + (a < 0.f) : lb;
    p.stat[cs_stat(n, CS_LQ)] = (float)(o2 - lse2 + ca);
  }
  // bf16: a row that takes no part is zero for the column pass, whose scores of it could pass fp32's range (the infinite
  // statistic takes a finite score out, not an infinite one; fp32's scores are of scaled values)
  if (NP == 1 && p.stat && lb < 0 && lane < LPR) *reinterpret_cast<u32x2*>(p.ximg + n * (2 * DP) + 2 * c) = u32x2{0, 0};
  if (!p.dx || lane >= LPR) return;
  const double il = L == 0. ? 0. : (NP == 2 ? 0x1p-14 : 1.) / L;  // fp32: O holds 2^14 times its items; L may pass fp32's range
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (c + j >= p.D) continue;
    float v = 0.f;
    if (lost) v = NAN;
    else if (lb >= 0) v = L == 0. ? 0.f : a * q * (NP == 2 ? (float)(o[j] * il) - wv[j] : o[j] * (float)il - wv[j]);
    else if (lb == -2) v = NAN;
    p.dx[n * p.D + c + j] = v;
  }
}

// The rows, and up to CS_TAIL_ROWS of them (one round of that workgroup's loads) the total in the grid's last
// workgroup. Forwards of 3000 x 64 to 100,000 x 128 items replayed from a graph: 0 to 1 us more than with a kernel
// of its own up to 2048 rows, 3 to 5 us more at 2500 and 4 to 13 at 8192. A call bound by the host gains its launch
// (64 rows: 19 us against 22).
constexpr int CS_TAIL_ROWS = 2048;
template <int DP, int NP, int NWV>
__global__ __launch_bounds__(NWV == 1 ? 256 : 64 * NWV) void cs_rows_kernel(CsRows p) {
  cs_row<DP, NP, NWV>(p);
  if (!p.done) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's row losses are out
  __syncthreads();
  if (ticket_last(p.done, blockIdx.x, gridDim.x)) cs_total(p);
}

// ---- backward ------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void cs_dx_kernel(const float* u, int64_t n, float scale, const CsScal* scal,
                                                    const float* gscale, void* out, int bf16) {
  cs_dx(blockIdx.x, 256, u, n, scale, scal, gscale, out, bf16);
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
    for (int s = 0; s < nsplit; ++s) M = fmaxf(M, m[v * nsplit + s]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < nsplit; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(O + (s * V + v) * DP + c);
    if constexpr (NP == 2) o += x * __builtin_amdgcn_exp2f(m[v * nsplit + s] - M);
    else o += x;
  }
  float f = scale * scal->inv_z * (gscale ? *gscale : 1.f);
  int ex = 0;
  if constexpr (NP == 2) {
    float frac;
    ex = cs_exp2_split(M, frac) - CS_XREF;
    f *= frac;
  }
  for (int j = 0; j < 4; ++j)
    if (c + j < D) {
      const float x = NP == 2 ? ldexpf(o[j] * f, ex) : o[j] * f;
      if (bf16) ((__bf16*)out)[v * D + c + j] = (__bf16)x;
      else ((float*)out)[v * D + c + j] = x;
    }
}

// ---- host ----------------------------------------------------------------------------------------
int cs_width(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// How a pass's resident blocks are spread: `full` of them whole, each of the others split into s streamed
// ranges, whichever costs least with `slots` workgroups at a time. A workgroup takes its tiles (5 TFLOP/s
// of matrix work a CU, measured) and 6 us to start and end; partials are written and read (4 TB/s).
// us, and bytes per us.
struct CsSpread {
  int full, s;
  int64_t per;
};
CsSpread cs_spread(int64_t nrb, int64_t tiles, const CsCfg& c, int D, int NP, int64_t rows, bool col) {
  const int64_t slots = 256 * c.WG, block = 16 * c.UB * c.NW;
  const double tile = (double)block * c.KT * D * 4 * (NP == 2 ? 3 : 1) * c.WG / 5e6;
  CsSpread best{0, 1, tiles};
  if (nrb < 1 || tiles < 1) return best;
  double best_cost = 1e300;
  // the column pass writes a whole block's gradient itself: whole rounds of blocks need no partials
  const int64_t fulls[3] = {0, nrb / slots * slots, nrb};
  for (int i = 0; i < (col ? 3 : 1); ++i) {
    const int64_t full = fulls[i], rest = nrb - full;
    if (i > 0 && full == fulls[i - 1]) continue;
    const double base = (double)ceil_div(full, slots) * (tiles * tile + 6.);
    const int64_t part = rows - full * block;
    // over the distinct splits, coarsest first
    for (int64_t per = tiles, s = 1; s <= 1024 && (s == 1 || rest * s <= 4 * slots);) {
      const double cost = base + (rest > 0 ? (double)ceil_div(rest * s, slots) * (per * tile + 6.) + part * s * D * 8. / 4e6 : 0.);
      if (cost < best_cost) {
        best_cost = cost;
        best = CsSpread{(int)full, (int)s, per};
      }
      if (per <= 1 || rest < 1) break;
      per = ceil_div(tiles, s + 1) < per ? ceil_div(tiles, s + 1) : per - 1;
      s = ceil_div(tiles, per);
    }
  }
  return best;
}

struct CsShape {
  int64_t N, Npad, V, Vpad, D;
  int DP, NP, es;
  bool wimage, few;
  int rsplit;
  CsSpread col;
  int64_t rtiles, rper, ctiles, rnrb, cnrb;
  int64_t prows;  // the column pass's rows with partials
};
CsShape cs_plan(int64_t N, int64_t V, int64_t D, int dtype, int want) {
  CsShape s;
  s.N = N;
  s.V = V;
  s.D = D;
  s.DP = cs_width(D);
  s.NP = dtype == RS_DTYPE_F32 ? 2 : 1;
  s.es = dtype == RS_DTYPE_F32 ? 4 : 2;
  s.Npad = (N + 63) / 64 * 64;
  s.Vpad = (V + 63) / 64 * 64;
  s.wimage = s.NP == 2 || D % 8 != 0;
  const CsCfg rc = cs_cfg(s.DP, s.NP, want & RS_CATALOG_DX ? CS_ROW : CS_STATS), cc = cs_cfg(s.DP, s.NP, CS_COL);
  s.rtiles = ceil_div(V, rc.KT);
  s.ctiles = s.Npad / cc.KT;
  s.rnrb = ceil_div(N, 16 * rc.UB * rc.NW);
  s.cnrb = ceil_div(V, 16 * cc.UB * cc.NW);
  const CsSpread row = cs_spread(s.rnrb, s.rtiles, rc, s.DP, s.NP, N, false);
  s.rsplit = row.s;
  s.col = cs_spread(s.cnrb, s.ctiles, cc, s.DP, s.NP, V, true);
  if (s.ctiles == 0) s.col.full = (int)s.cnrb;  // no rows: every gradient is the whole blocks' zero
  s.prows = V - (int64_t)s.col.full * 16 * cc.UB * cc.NW;
  if (s.prows < 0) s.prows = 0;
  // few rows, loss alone, fp32: cs_few_kernel, three workgroups a CU
  s.few = s.NP == 2 && want == 0 && D % 4 == 0 && N <= (s.DP == 256 ? 32 : 64);
  if (s.few && N) {
    s.rtiles = ceil_div(V, 64);
    s.rsplit = (int)(s.rtiles < 768 ? s.rtiles : 768);
    s.wimage = false;
  }
  s.rper = ceil_div(s.rtiles, s.rsplit);
  return s;
}
// the plan of the sizes, kept from one call for the next of equal sizes (a forward and its backward; the
// search takes 1 to 4 us of the host's time)
const CsShape& cs_shape(int64_t N, int64_t V, int64_t D, int dtype, int want) {
  struct Last {
    int64_t N, V, D;
    int dtype, want;
    CsShape s;
  };
  static thread_local Last last{-1, 0, 0, 0, 0, {}};
  if (last.N != N || last.V != V || last.D != D || last.dtype != dtype || last.want != want)
    last = Last{N, V, D, dtype, want, cs_plan(N, V, D, dtype, want)};
  return last.s;
}

struct CsKeep {
  CsScal* scal;
  char *ximg, *wimg;
  int32_t* lab;
  float *kx, *wstat, *stat, *dx;
  bool ok;
  size_t bytes;
  CsKeep(void* base, size_t size, const CsShape& s, int want) {
    Carve c(base, size);
    scal = c.take<CsScal>(1);
    ximg = c.take<char>((size_t)s.Npad * s.DP * 2 * s.NP);
    wimg = s.wimage ? c.take<char>((size_t)s.V * s.DP * 2 * s.NP) : nullptr;
    lab = c.take<int32_t>(s.Npad);
    kx = c.take<float>(s.Npad);
    wstat = s.wimage && s.NP == 2 ? c.take<float>(s.Vpad * 3) : nullptr;
    stat = c.take<float>(s.Npad * 4);
    dx = want & RS_CATALOG_DX ? c.take<float>((size_t)s.N * s.D) : nullptr;
    bytes = align_up(c.off, 256);
    ok = c.ok();
  }
};
struct CsFwdWs {
  unsigned int* done;
  float *m, *O;
  double* l;
  bool ok;
  size_t bytes;
  CsFwdWs(void* base, size_t size, const CsShape& s, int want) {
    Carve c(base, size);
    done = c.take<unsigned int>(TICKET_WORDS);
    m = c.take<float>((size_t)s.rsplit * s.N);
    l = c.take<double>((size_t)s.rsplit * s.N);
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
    const size_t part = want & RS_CATALOG_DW ? (size_t)s.col.s * s.prows : 0;
    m = c.take<float>(part);
    O = c.take<float>(part * s.DP);
    bytes = align_up(c.off, 256);
    ok = c.ok();
  }
};

template <int MODE>
void cs_launch_pass(const CsShape& s, const CsPass& p, int64_t grid, hipStream_t st) {
#define CS_GO(WD, PL) \
  if (s.DP == WD && s.NP == PL) \
    hipLaunchKernelGGL((cs_pass_kernel<WD, PL, MODE>), dim3((unsigned)grid), dim3(64 * cs_cfg(WD, PL, MODE).NW), 0, st, p);
  CS_GO(64, 1) CS_GO(64, 2) CS_GO(128, 1) CS_GO(128, 2) CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
}

int cs_check(int64_t N, int64_t V, int64_t D, int dtype, float scale, int want, const char* what) {
  RS_REQUIRE(N >= 0 && V >= 1 && D >= 1, "%s: bad sizes N=%lld V=%lld D=%lld", what, (long long)N, (long long)V,
             (long long)D);
  // labels in 31 bits; grids below 2^32 threads: the row join's 64 a row, the column pass's 4 an item at most,
  // with one for 4 values of x
  RS_REQUIRE(N < (1ll << 26) && V < (1ll << 29), "%s: N must be below 2^26, V below 2^29", what);
  RS_REQUIRE(N * D < (1ll << 33), "%s: X must hold fewer than 2^33 values", what);
  RS_REQUIRE(dtype == RS_DTYPE_F32 || dtype == RS_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
  RS_REQUIRE(scale >= 0x1p-60f && scale <= 0x1p60f, "%s: scale must lie between 2^-60 and 2^60", what);
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
  return CsKeep(nullptr, 0, cs_shape(N, V, D, dtype, want), want).bytes;
}

extern "C" size_t rs_catalog_softmax_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype, int want) {
  if (cs_check(N, V, D, dtype, 1.f, want, "catalog_softmax") != RS_OK) return 0;
  const CsShape& s = cs_shape(N, V, D, dtype, want);
  const size_t a = CsFwdWs(nullptr, 0, s, want).bytes, b = CsBwdWs(nullptr, 0, s, want).bytes;
  return a > b ? a : b;
}

extern "C" int rs_catalog_softmax_fwd(const void* X, const void* W, const int64_t* labels, const float* weights,
                                      int64_t N, int64_t V, int64_t D, int dtype, float scale, int64_t ignore_index,
                                      int mean, int want, float* loss, float* row_loss, float* lse, void* keep,
                                      size_t keep_bytes, void* workspace, size_t workspace_bytes, rs_stream_t stream) {
  const int rc = cs_check(N, V, D, dtype, scale, want, "catalog_softmax_fwd");
  if (rc != RS_OK) return rc;
  RS_REQUIRE(W && loss && keep && workspace && (N == 0 || (X && labels && row_loss)),
             "catalog_softmax_fwd: null pointer");
  RS_REQUIRE(aligned16(X) && aligned16(W) && aligned16(keep) && aligned16(workspace),
             "catalog_softmax_fwd: X, W, keep and workspace must be 16-byte aligned");
  const CsShape& s = cs_shape(N, V, D, dtype, want);
  const CsKeep k(keep, keep_bytes, s, want);
  const CsFwdWs w(workspace, workspace_bytes, s, want);
  if (!k.ok || !w.ok) {
    set_error("catalog_softmax_fwd: %s too small", k.ok ? "workspace" : "keep buffer");
    return RS_ERR_WORKSPACE;
  }
  hipStream_t st = as_stream(stream);
  const float kbase = (float)((double)scale * CS_LOG2E);
  if (N > 0 && s.few) {
    const CsFew f{(const float*)X, (const float*)W, labels, N, V, D, ignore_index, s.rtiles, kbase, k.lab, w.m, w.l, w.done};
    const int Q = (int)ceil_div(N, 16);
#define CS_GO(WD, QQ)                                          \
  if (s.DP == WD && (Q == QQ || (QQ == 4 && Q == 3)))          \
    hipLaunchKernelGGL((cs_few_kernel<WD, QQ>), dim3(s.rsplit), dim3(256), 0, st, f);
    CS_GO(64, 1) CS_GO(64, 2) CS_GO(64, 4) CS_GO(128, 1) CS_GO(128, 2) CS_GO(128, 4)
    CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
  } else if (N > 0) {
    const int rpb = 256 / (s.DP / 4);
    CsImage im{X, W, k.ximg, k.wimg, N, s.Npad, V, s.Vpad, D, s.Npad * s.DP * 2, V * s.DP * 2, ignore_index, labels, k.lab,
               k.kx, k.wstat, k.scal, w.done, 0};
    int64_t xb = ceil_div(s.Npad, rpb), wb = s.wimage ? ceil_div(s.NP == 2 ? s.Vpad : V, rpb) : 0;
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
    p.t_plane = s.NP == 2 ? V * s.DP * 2 : 0;
    p.r_ld = s.DP * 2;
    p.t_ld = s.wimage ? s.DP * 2 : D * 2;
    p.r_ch = s.DP / 8;
    p.t_ch = (int)(p.t_ld / 16);
    p.zero = (const char*)k.scal->zero;
    p.nsplit = s.rsplit;
    p.tiles = s.rtiles;
    p.per = s.rper;
    p.nrb = (int)s.rnrb;
    p.pR = N;
    p.scal = k.scal;
    p.scale = scale;
    p.kbase = kbase;
    p.kr = k.kx;
    p.stat = k.wstat;
    p.lab = k.lab;
    p.m = w.m;
    p.l = w.l;
    p.O = w.O;
    if (want & RS_CATALOG_DX) cs_launch_pass<CS_ROW>(s, p, s.rnrb * s.rsplit, st);
    else cs_launch_pass<CS_STATS>(s, p, s.rnrb * s.rsplit, st);
  }
  const CsRows r{X, W, s.NP == 1, N, s.Npad, V, D, s.rsplit, w.m, w.O, w.l, k.lab, weights, k.kx, scale, kbase, row_loss,
                 lse, k.dx, want & RS_CATALOG_DW ? k.stat : nullptr, k.ximg, k.scal,
                 N <= CS_TAIL_ROWS ? w.done : nullptr, mean, loss};
  if (N > 0) {
    // many splits of few rows: a workgroup per row, else a wave
    const int wide = s.rsplit > 64 ? 8 : s.rsplit > 8 ? 4 : 0;
    const dim3 gr((unsigned)(wide ? s.Npad : s.Npad / 4));
#define CS_GO(WD, PL)                                                                                     \
  if (s.DP == WD && s.NP == PL) {                                                                         \
    if (wide == 8) hipLaunchKernelGGL((cs_rows_kernel<WD, PL, 8>), gr, dim3(512), 0, st, r);              \
    else if (wide == 4) hipLaunchKernelGGL((cs_rows_kernel<WD, PL, 4>), gr, dim3(256), 0, st, r);         \
    else hipLaunchKernelGGL((cs_rows_kernel<WD, PL, 1>), gr, dim3(256), 0, st, r);                        \
  }
    CS_GO(64, 1) CS_GO(64, 2) CS_GO(128, 1) CS_GO(128, 2) CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
  }
  if (N == 0 || !r.done) hipLaunchKernelGGL(cs_total_kernel, dim3(1), dim3(1024), 0, st, r);
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
  const CsShape& s = cs_shape(N, V, D, dtype, want);
  const CsKeep k(const_cast<void*>(keep), keep_bytes, s, want);
  const CsBwdWs w(workspace, workspace_bytes, s, want);
  if (!k.ok || !w.ok) {
    set_error("catalog_softmax_bwd: %s too small", k.ok ? "workspace" : "keep buffer");
    return RS_ERR_WORKSPACE;
  }
  hipStream_t st = as_stream(stream);
  if (dX && N > 0 && !dW)
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
    p.r_ld = s.wimage ? s.DP * 2 : D * 2;
    p.t_ld = s.DP * 2;
    p.r_ch = (int)(p.r_ld / 16);
    p.t_ch = s.DP / 8;
    p.zero = (const char*)k.scal->zero;
    p.nsplit = s.col.s;
    p.full = s.col.full;
    p.pR = s.prows;
    p.tiles = s.ctiles;
    p.per = s.col.per;
    p.nrb = (int)s.cnrb - s.col.full;
    p.scal = k.scal;
    p.scale = scale;
    p.kbase = (float)((double)scale * CS_LOG2E);
    p.kr = k.wstat;
    p.stat = k.stat;
    p.m = w.m;
    p.O = w.O;
    p.out = dW;
    p.ld = D;
    p.out_bf16 = s.NP == 1;
    p.gscale = gscale;
    int64_t grid = p.full + (int64_t)p.nrb * p.nsplit;
    if (dX && N > 0) {
      p.dx_unit = k.dx;
      p.n_dx = N * D;
      p.dx = dX;
      grid += ceil_div(N * D, 256 * cs_cfg(s.DP, s.NP, CS_COL).NW);
    }
    cs_launch_pass<CS_COL>(s, p, grid, st);
    if (s.prows > 0) {
      void* out = (char*)dW + (V - s.prows) * D * s.es;
      const dim3 gd((unsigned)ceil_div(s.prows, 256 / (s.DP / 4)));
#define CS_GO(WD, PL)                                                                                                \
  if (s.DP == WD && s.NP == PL)                                                                                     \
    hipLaunchKernelGGL((cs_dw_kernel<WD, PL>), gd, dim3(256), 0, st, w.m, w.O, s.col.s, s.prows, D, scale, k.scal,  \
                       gscale, out, s.NP == 1);
      CS_GO(64, 1) CS_GO(64, 2) CS_GO(128, 1) CS_GO(128, 2) CS_GO(256, 1) CS_GO(256, 2)
#undef CS_GO
    }
  }
  return check_launch("catalog_softmax_bwd");
}
