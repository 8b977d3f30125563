// GELU whose input is kept for the backward pass in 8 bits (gfx950).
//
//   forward    y = x Phi(x);  kept = MX e4m3 of x: per 32 values a scale 2^e, the smallest with
//              amax / 2^e <= 448, and x / 2^e rounded to e4m3 (nearest, ties to even)
//   backward   x~ = the kept value;  dx = dy (Phi(x~) + x~ phi(x~)),  again = x~ Phi(x~) on request (the
//              second linear layer's weight gradient needs the activation, which then need not be kept)
//
// Phi is the normal distribution's cdf (the erf form of GELU), phi its density.  Both directions read and
// write each value once and are bound by HBM: 16 B of bf16 a lane and load, four lanes share a block.
// 18464 x 4096, calls one after the other: 68.5 us forward (5.6 TB/s, part of it from the last-level cache; a copy of 2 GiB
// reaches 4.9), 92 us backward with `again` (5.8 TB/s), 72 us without (5.3 TB/s; the vector unit counts too: two more operations
// a value are 3 %).  What it took: no infinity tests on the usual path (167 -> 159 us for both).
#include "common.h"
#include "mx.h"

namespace i2pc {
namespace gelu8 {

// Phi(-|x|) = t P(t) ex with ex = exp(-x^2 / 2) and t = 1 / (1 + 0.29 |x|): Phi(-|x|) / ex is a smooth function of t down to
// t = 0, where it goes as 1 / |x|.  P is a minimax fit of degree 5 over |x| <= 14, made for this kernel, of the error over the
// smaller of 5e-8 and 2^-13 Phi(-|x|): the tail is within 5.8e-8 and within 2^-13 of its own size, so that GELU and its slope
// hold bf16's rounding far below zero too (down to x = -13, where ex leaves fp32's normal range).
__device__ __forceinline__ float normal_tail(float x, float& ex) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.29f, fabsf(x), 1.0f));
  ex = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
  float p = fmaf(t, -0.08956327289f, 0.2875475585f);
  p = fmaf(t, p, -0.09686156362f);
  p = fmaf(t, p, 0.1819336414f);
  p = fmaf(t, p, 0.09999677539f);
  p = fmaf(t, p, 0.1169468239f);
  return p * t * ex;
}
// GELU(x) = max(x, 0) - |x| Phi(-|x|).  ENDS: +-inf may come in (inf * 0 otherwise).  NaN stays NaN in both forms.
template <bool ENDS>
__device__ __forceinline__ float gelu(float x, float tail) {
  const float y = fmaf(-fabsf(x), tail, fmaxf(x, 0.f));
  return ENDS && fabsf(x) == INFINITY ? fmaxf(x, 0.f) : y;
}
// Phi(x) + x phi(x).  Below zero Phi is the tail itself: by way of 1 or 1 / 2 the error of those would stay.
template <bool ENDS>
__device__ __forceinline__ float gelu_slope(float x, float tail, float ex) {
  const float c = x < 0.f ? tail : 1.0f - tail;
  return ENDS && fabsf(x) == INFINITY ? c : fmaf(x * 0.39894228040143268f, ex, c);
}

// x / 2^e within e4m3's range, which only infinities of a block of scale 2^127 leave
__device__ __forceinline__ float within(float v) { return v != v ? v : fminf(fmaxf(v, -448.f), 448.f); }

__device__ __forceinline__ float lo16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// where chunk c (8 values) of a [rows][dim] array with row pitch ld starts
__device__ __forceinline__ int64_t at(uint32_t c, uint32_t per_row, int64_t ld) {
  const uint32_t r = c / per_row;
  return r * ld + (int64_t)(c - r * per_row) * 8;
}

__global__ __launch_bounds__(256) void k_gelu_keep(const uint16_t* x, int64_t ldx, uint32_t chunks, uint32_t per_row, uint16_t* y, int64_t ldy, uint8_t* __restrict__ kept,
                                                   uint8_t* __restrict__ scale) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  // chunks is a multiple of four: a block's four lanes are on or off together
  if (c >= chunks) return;
  const uint4 w = *reinterpret_cast<const uint4*>(x + at(c, per_row, ldx));
  const float v[8] = {lo16(w.x), hi16(w.x), lo16(w.y), hi16(w.y), lo16(w.z), hi16(w.z), lo16(w.w), hi16(w.w)};
  float am = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) am = fmaxf(am, fabsf(v[j]));
  am = fmaxf(am, __shfl_xor(am, 1));
  am = fmaxf(am, __shfl_xor(am, 2));
  const int e = mx::mx_exponent(am);
  const float mul = mx::exp2i(-e);
  float q[8], g[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float ex;
    const float tail = normal_tail(v[j], ex);
    q[j] = v[j] * mul;
    g[j] = gelu<false>(v[j], tail);
  }
  if (__builtin_expect(am == INFINITY, 0)) {
    asm volatile("");                                  // a branch, not selects: hardly ever taken
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float ex;
      const float tail = normal_tail(v[j], ex);
      q[j] = within(v[j] * mul);
      g[j] = gelu<true>(v[j], tail);
    }
  }
  int d0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false), d1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
  d0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], d0, true);
  d1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], d1, true);
  *reinterpret_cast<uint4*>(y + at(c, per_row, ldy)) =
      make_uint4(pk2bf(g[0], g[1]), pk2bf(g[2], g[3]), pk2bf(g[4], g[5]), pk2bf(g[6], g[7]));
  *reinterpret_cast<int2*>(kept + (int64_t)c * 8) = make_int2(d0, d1);
  if ((c & 3) == 0) scale[c >> 2] = (uint8_t)(e + 127);
}

template <bool AGAIN>
__global__ __launch_bounds__(256) void k_gelu_back(const uint16_t* dy, int64_t lddy, const uint8_t* __restrict__ kept,
                                                   const uint8_t* __restrict__ scale, uint32_t chunks, uint32_t per_row,
                                                   uint16_t* dx, int64_t lddx, uint16_t* __restrict__ again,
                                                   int64_t lda) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= chunks) return;
  const uint4 w = *reinterpret_cast<const uint4*>(dy + at(c, per_row, lddy));
  const int2 k = *reinterpret_cast<const int2*>(kept + (int64_t)c * 8);
  const int e = scale[c >> 2];
  const float mul = mx::exp2i(e - 127);
  const float d[8] = {lo16(w.x), hi16(w.x), lo16(w.y), hi16(w.y), lo16(w.z), hi16(w.z), lo16(w.w), hi16(w.w)};
  float x[8], g[8], a[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int word = h ? k.y : k.x;
    const auto p0 = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), p1 = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
    x[4 * h] = p0[0] * mul, x[4 * h + 1] = p0[1] * mul, x[4 * h + 2] = p1[0] * mul, x[4 * h + 3] = p1[1] * mul;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float ex;
    const float tail = normal_tail(x[j], ex);
    a[j] = gelu<false>(x[j], tail);
    g[j] = d[j] * gelu_slope<false>(x[j], tail, ex);
  }
  if (__builtin_expect(e >= 127 + 120, 0)) {           // 448 * 2^120 is above the largest float
    asm volatile("");                                  // a branch, not selects
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float ex;
      const float tail = normal_tail(x[j], ex);
      a[j] = gelu<true>(x[j], tail);
      g[j] = d[j] * gelu_slope<true>(x[j], tail, ex);
    }
  }
  *reinterpret_cast<uint4*>(dx + at(c, per_row, lddx)) =
      make_uint4(pk2bf(g[0], g[1]), pk2bf(g[2], g[3]), pk2bf(g[4], g[5]), pk2bf(g[6], g[7]));
  if constexpr (AGAIN)
    *reinterpret_cast<uint4*>(again + at(c, per_row, lda)) =
        make_uint4(pk2bf(a[0], a[1]), pk2bf(a[2], a[3]), pk2bf(a[4], a[5]), pk2bf(a[6], a[7]));
}

inline bool aligned(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

}  // namespace gelu8
}  // namespace i2pc

using namespace i2pc;

static int gelu8_shape(const char* what, int64_t rows, int dim) {
  I2PC_REQUIRE(rows >= 0 && dim > 0 && dim % 32 == 0, "%s: dim=%d must be a positive multiple of 32", what, dim);
  // 32-bit chunk indexes, and a grid of 256-thread workgroups over them
  if (rows * (dim / 8) >= (int64_t)1 << 31)
    return set_error(I2PC_EUNSUPPORTED, "%s: %lld rows of %d values are above 2^34 values", what, (long long)rows, dim);
  return I2PC_OK;
}

extern "C" int i2pc_gelu_fp8(const void* x, int64_t ldx, int64_t rows, int dim, void* y, int64_t ldy, void* kept,
                             void* kept_scale, void* stream) {
  clear_error();
  if (const int rc = gelu8_shape("gelu_fp8", rows, dim)) return rc;
  if (rows == 0) return I2PC_OK;
  I2PC_REQUIRE(x && y && kept && kept_scale, "NULL pointer");
  I2PC_REQUIRE(ldx >= dim && ldy >= dim && gelu8::aligned(x, ldx) && gelu8::aligned(y, ldy) && gelu8::aligned(kept, 0),
               "gelu_fp8: rows of at least dim values, 16-byte aligned (pitch a multiple of 8)");
  const uint32_t per_row = dim / 8, chunks = (uint32_t)(rows * per_row);
  hipLaunchKernelGGL(gelu8::k_gelu_keep, dim3((chunks + 255) / 256), dim3(256), 0, as_stream(stream),
                     static_cast<const uint16_t*>(x), ldx, chunks, per_row, static_cast<uint16_t*>(y), ldy,
                     static_cast<uint8_t*>(kept), static_cast<uint8_t*>(kept_scale));
  return check_launch("gelu_fp8");
}

extern "C" int i2pc_gelu_fp8_backward(const void* dy, int64_t lddy, const void* kept, const void* kept_scale, int64_t rows,
                                      int dim, void* dx, int64_t lddx, void* again, int64_t ld_again, void* stream) {
  clear_error();
  if (const int rc = gelu8_shape("gelu_fp8_backward", rows, dim)) return rc;
  if (rows == 0) return I2PC_OK;
  I2PC_REQUIRE(dy && kept && kept_scale && dx, "NULL pointer");
  I2PC_REQUIRE(lddy >= dim && lddx >= dim && (!again || ld_again >= dim) && gelu8::aligned(dy, lddy) &&
                   gelu8::aligned(dx, lddx) && gelu8::aligned(kept, 0) && (!again || gelu8::aligned(again, ld_again)),
               "gelu_fp8_backward: rows of at least dim values, 16-byte aligned (pitch a multiple of 8)");
  const uint32_t per_row = dim / 8, chunks = (uint32_t)(rows * per_row);
  const dim3 grid((chunks + 255) / 256), block(256);
  if (again)
    hipLaunchKernelGGL(gelu8::k_gelu_back<true>, grid, block, 0, as_stream(stream), static_cast<const uint16_t*>(dy), lddy,
                       static_cast<const uint8_t*>(kept), static_cast<const uint8_t*>(kept_scale), chunks, per_row,
                       static_cast<uint16_t*>(dx), lddx, static_cast<uint16_t*>(again), ld_again);
  else
    hipLaunchKernelGGL(gelu8::k_gelu_back<false>, grid, block, 0, as_stream(stream), static_cast<const uint16_t*>(dy), lddy,
                       static_cast<const uint8_t*>(kept), static_cast<const uint8_t*>(kept_scale), chunks, per_row,
                       static_cast<uint16_t*>(dx), lddx, nullptr, 0);
  return check_launch("gelu_fp8_backward");
}
