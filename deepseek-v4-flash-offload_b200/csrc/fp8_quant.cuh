// E4M3 quantisation of one block of 128 columns: the arithmetic shared by
// act_quant (fp8_quant.cu) and the product that quantises its own rows
// (fp8_matmul.cu), so that both give the same codes.
//
// With a = max(1e-4, max |x|) of the block:
//   power-of-two scales: s = 2^e with the smallest e that gives a <= 448 2^e,
//     q = e4m3(x 2^-e) (the division is exact, so q has one rounding);
//   fp32 scales: s = a / 448, q = the E4M3 value nearest to the real 448 x / a.
//     The quotient is the product with the block's reciprocal, corrected once
//     by its remainder (Markstein 1990), and then less than one step of fp32
//     from the real one.  For 16-bit x (0.875 x is exact) a quotient is a tie
//     of E4M3 or more than 2^-20 away from one, so rounding it gives the
//     nearest code.  For fp32 x the remainder takes in what 0.875 x lost, and
//     a quotient that comes out as a tie is moved off it by one step where its
//     own remainder, exact there, is not 0.  A division per element was the
//     limit: 27.8 us instead of 21.4 for 8192 x 4096 bf16.
// A NaN stays NaN and leaves its block's scale alone; an infinity takes the
// largest finite value's scale and saturates.
#pragma once

#include "common.cuh"

namespace dsv4 {

// Smallest e with a <= 448 * 2^e (448 = 1.75 * 2^8), a normal and finite.
__device__ __forceinline__ int scale_exp_448(float a) {
  const uint32_t u = __float_as_uint(a);
  return (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// 0.875 x / d with r = 1 / d rounded to nearest; infinities and NaN as 0.875 x r.
// WIDE: x has more than 16 bits.
template <bool WIDE>
__device__ __forceinline__ float fp8_quotient(float x, float d, float r) {
  const float n = 0.875f * x, q = n * r;
  const float rem = WIDE ? fmaf(-q, d, n) + fmaf(0.875f, x, -n) : fmaf(-q, d, n);
  return fabsf(q) < 1e30f ? fmaf(rem, r, q) : q;
}
// E4M3 values and ties have at most five significant bits.
__device__ __forceinline__ bool fp8_maybe_tie(float q) { return (__float_as_int(q) & 0x7ffff) == 0; }
// q moved by one step towards the real 0.875 x / d, if that is another number.
__device__ __forceinline__ float fp8_off_tie(float q, float x, float d) {
  const float n = 0.875f * x, rem = fmaf(-q, d, n) + fmaf(0.875f, x, -n);
  if (rem == 0.f || !(fabsf(q) < 1e30f)) return q;
  return __int_as_float(__float_as_int(q) + ((__float_as_int(rem) ^ __float_as_int(q)) < 0 ? -1 : 1));
}
// The block's a over the 16 lanes that hold it, eight columns each.
__device__ __forceinline__ float fp8_amax(const float (&v)[8]) {
  float a = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = fmaxf(a, fabsf(v[j]));   // fmaxf drops a NaN
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  return fminf(fmaxf(a, 1e-4f), 3.402823466e+38f);
}
// A lane's eight codes (byte j = column j) with power-of-two scales 2^e ...
__device__ __forceinline__ uint2 fp8_codes_pow2(const float (&v)[8], int e) {
  const float inv = pow2i(-e);
  return make_uint2(e4m3x2(v[0] * inv, v[1] * inv) | (e4m3x2(v[2] * inv, v[3] * inv) << 16),
                    e4m3x2(v[4] * inv, v[5] * inv) | (e4m3x2(v[6] * inv, v[7] * inv) << 16));
}
// ... and with the scale a / 448: 448 x / a = (0.875 x) / (a / 512), a / 512 exact.
template <bool WIDE>
__device__ __forceinline__ uint2 fp8_codes_fp32(const float (&v)[8], float a) {
  const float d = a * 0.001953125f, r = __frcp_rn(d);
  float q[8];
  bool tie = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    q[j] = fp8_quotient<WIDE>(v[j], d, r);
    if constexpr (WIDE) tie |= fp8_maybe_tie(q[j]);
  }
  if (WIDE && tie) {   // one element in 2^19, and zeros
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (fp8_maybe_tie(q[j])) q[j] = fp8_off_tie(q[j], v[j], d);
  }
  return make_uint2(e4m3x2(q[0], q[1]) | (e4m3x2(q[2], q[3]) << 16), e4m3x2(q[4], q[5]) | (e4m3x2(q[6], q[7]) << 16));
}
__device__ __forceinline__ float fp8_scale_fp32(float a) { return __fdiv_rn(a, 448.f); }

}  // namespace dsv4
