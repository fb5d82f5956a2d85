// Products of 8-bit integers: what their kernels share.
//
//   most[t] = max |x[t]|,  q[t] = rint(x[t] * (127 / most[t])),  y[t, n] = (sum q[t] w[n]) * (most[t] / 127) * scale[n]
//
// with whole sums in 32 bits (|sum| <= 127 * 127 * K) and everything else in float32. A row of magnitudes under 2^-100 has
// codes of 0 (its factor 127 / most would pass float32's range); a row that holds an infinity or a NaN becomes NaN.
// Rows are held padded with zeros to whole stages of 128 columns ("width"), which add nothing to a sum.
#pragma once
#include "common.h"

typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int INT8_STAGE = 128;
constexpr int INT8_MOST_WIDTH = 1 << 17;  // 127 * 127 * 2^17 < 2^31

struct IntProducts {
  typedef i32x4_t Operand;
  typedef i32x4_t Sums;
  static __device__ __forceinline__ Sums add(Operand w, Operand a, Sums c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, a, c, 0, 0, 0); }
};

// The magnitude's bits, whose order is the numbers' and puts NaN above all.
__device__ __forceinline__ unsigned magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ unsigned wave_max_bits(unsigned m) {
  // whole numbers as the bits of non-negative floats: the larger of either is the larger of both, but for NaN's, which are told apart first
  const bool nan = m > 0x7f800000u;
  const unsigned r = __float_as_uint(wave_max(__uint_as_float(nan ? 0u : m)));
  return __builtin_amdgcn_ballot_w64(nan) != 0 ? 0x7fc00000u : r;
}
__device__ __forceinline__ float code_factor(unsigned most) {
  return most >= 0x0d800000u && most < 0x7f800000u ? 127.0f / __uint_as_float(most) : 0.0f;  // 2^-100
}
__device__ __forceinline__ float row_scale_of(unsigned most) {
  return most < 0x7f800000u ? __uint_as_float(most) / 127.0f : __uint_as_float(0x7fc00000u);
}
// Four codes in a word. The sum with 1.5 * 2^23 rounds the product to a whole number, to even where two are as near, and leaves it
// in the low byte; the product is rounded to float32 before, not fused with the sum: codes are then the same however they are made.
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d, float by) {
#pragma clang fp contract(off)
  const float pa = a * by, pb = b * by, pc = c * by, pd = d * by;
  const unsigned ua = __float_as_uint(pa + 12582912.0f), ub = __float_as_uint(pb + 12582912.0f);
  const unsigned uc = __float_as_uint(pc + 12582912.0f), ud = __float_as_uint(pd + 12582912.0f);
  const unsigned ab = __builtin_amdgcn_perm(ub, ua, 0x0c0c0400), cd = __builtin_amdgcn_perm(ud, uc, 0x04000c0c);
  return ab | cd;
}

int int8_tiles(const void* a, const float* a_scale, const void* w, const float* w_scale, void* c, int out_dtype, int M, int N, int width, int tile,
               int parts, int act_kind, float limit, hipStream_t stream);
