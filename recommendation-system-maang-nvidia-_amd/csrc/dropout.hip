// dropout.hip — dropout whose mask is a function of (seed, step, element) and is never stored: the
// forward and the backward make it from the same words, so a layer keeps 16 bytes instead of a mask.
//
// Words: Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011), key =
// the 64-bit seed, counter = (element / 4, step), word element % 4. Element i is kept iff its word is
// at least round(rate 2^32): y = x f, f = 1 / (1 - rate) rounded to fp32 and the product once more (then once
// to bf16); a dropped element is 0 whatever x holds there.
//
// Bound: HBM, one read and one write per element.
#include "split.hpp"

#include <cmath>

namespace rs {
namespace {

// four words of one counter; the 32 x 32 -> 64 products are one v_mad_u64_u32 each
__device__ __forceinline__ void do_philox(uint64_t ctr, uint64_t step, uint64_t key, uint32_t (&w)[4]) {
  uint32_t c0 = (uint32_t)ctr, c1 = (uint32_t)(ctr >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

// 8 elements (two counters) per thread; VEC: 16-byte accesses
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const void* __restrict__ x, int64_t n, uint32_t thr, float f,
                                                      const int64_t* __restrict__ ticket, void* __restrict__ y) {
  const uint64_t key = (uint64_t)ticket[0], step = (uint64_t)ticket[1];
  const int64_t i0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i0 >= n) return;
  const bool whole = VEC && i0 + 8 <= n;
  float v[8];
  if (whole) {
    if constexpr (BF16) {
      const u32x4 q = *reinterpret_cast<const u32x4*>((const __bf16*)x + i0);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = ib_lo(q[j]), v[2 * j + 1] = ib_hi(q[j]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 q = *reinterpret_cast<const f32x4*>((const float*)x + i0 + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * h + j] = q[j];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = 0.f;
      if (i0 + j < n) v[j] = BF16 ? (float)((const __bf16*)x)[i0 + j] : ((const float*)x)[i0 + j];
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[4];
    do_philox((uint64_t)i0 / 4 + h, step, key, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * h + j] = w[j] >= thr ? v[4 * h + j] * f : 0.f;
  }
  if (whole) {
    if constexpr (BF16) {
      *reinterpret_cast<u32x4*>((__bf16*)y + i0) =
          u32x4{ib_pk(v[0], v[1]), ib_pk(v[2], v[3]), ib_pk(v[4], v[5]), ib_pk(v[6], v[7])};
    } else {
      *reinterpret_cast<f32x4*>((float*)y + i0) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>((float*)y + i0 + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j < n) {
        if constexpr (BF16) ((__bf16*)y)[i0 + j] = (__bf16)v[j];
        else ((float*)y)[i0 + j] = v[j];
      }
  }
}

__global__ void dropout_ticket_kernel(int64_t* state, int64_t* ticket) {
  ticket[0] = state[0];
  ticket[1] = state[1];
  state[1] = (int64_t)((uint64_t)state[1] + 1u);
}

}  // namespace
}  // namespace rs

using namespace rs;

extern "C" int rs_dropout(const void* x, int64_t n, int dtype, double rate, const int64_t* ticket, void* y,
                          rs_stream_t stream) {
  RS_REQUIRE(n >= 0, "dropout: bad size %lld", (long long)n);
  RS_REQUIRE(dtype == RS_DTYPE_F32 || dtype == RS_DTYPE_BF16, "dropout: unknown dtype %d", dtype);
  RS_REQUIRE(rate >= 0. && rate < 1., "dropout: rate must lie in [0, 1), got %g", rate);
  const double thr = nearbyint(rate * 4294967296.);
  RS_REQUIRE(thr < 4294967296., "dropout: rate %.12g keeps no element of 2^32", rate);
  if (n == 0) return RS_OK;
  RS_REQUIRE(x && y && ticket, "dropout: null pointer");
  RS_REQUIRE(n < (1ll << 35) - 2048, "dropout: %lld elements are 2^35 or more", (long long)n);  // 2^32 threads
  const dim3 grid((unsigned)ceil_div(n, 2048));
  const float f = (float)(1. / (1. - rate));
  const bool vec = aligned16(x) && aligned16(y);
#define DO_GO(B, A)                                                                                           \
  if ((dtype == RS_DTYPE_BF16) == B && vec == A)                                                              \
    hipLaunchKernelGGL((dropout_kernel<B, A>), grid, dim3(256), 0, as_stream(stream), x, n, (uint32_t)thr, f, \
                       ticket, y);
  DO_GO(true, true) DO_GO(true, false) DO_GO(false, true) DO_GO(false, false)
#undef DO_GO
  return check_launch("dropout");
}

extern "C" int rs_dropout_ticket(int64_t* state, int64_t* ticket, rs_stream_t stream) {
  RS_REQUIRE(state && ticket && state != ticket, "dropout_ticket: null or shared pointers");
  hipLaunchKernelGGL(dropout_ticket_kernel, dim3(1), dim3(1), 0, as_stream(stream), state, ticket);
  return check_launch("dropout_ticket");
}
