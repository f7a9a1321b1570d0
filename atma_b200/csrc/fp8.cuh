// Rows in 8 bits: e4m3 values with an fp32 scale for every 128 channels.
//   s = max(max |x| / 448, 2^-126),  q = e4m3(x / s): what stands there is q s.
// The largest value of a block lands on 448, e4m3's largest, so that nothing saturates; the lower bound keeps x / s finite for blocks
// of zeros and of values that an fp32 quotient by 448 would flush.  A NaN or an infinity in a block makes its scale a NaN: every result
// that such a row takes part in is one.
// Rows that are given (fp8_four, fp8_one): the quotient is rounded once, to e4m3.  16-bit values over a largest one of their kind lie on, or
// nearly on, borders between two e4m3 values in numbers (in one block of seven or so), and a quotient that is rounded to fp32 in between
// lands on the border itself.  Results of fp32 arithmetic (.._times): a product with 1 / s, which is off by as little as they are.
#pragma once

#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace atma {

constexpr int kFp8Block = 128;
constexpr float kFp8Top = 448.0f, kFp8Least = 1.17549435e-38f;

__device__ __forceinline__ float max_nan(float a, float b) {                       // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// The correctly rounded quotient (checked for every mantissa; exponents only shift it), with one fma to correct a product.
__device__ __forceinline__ float fp8_scale(float largest) {
  constexpr float kInverse = 1.0f / kFp8Top;
  const float q = largest * kInverse;
  return max_nan(fmaf(fmaf(-q, kFp8Top, largest), kInverse, q), kFp8Least);
}
__device__ __forceinline__ float fp8_inverse(float s) { return __fdividef(1.0f, s); }          // to a unit in the last place; s is 2^-126 to 2^120

// x / s, rounded to odd; inv = 1 / s to a unit or two in the last place.
__device__ __forceinline__ float fp8_quotient(float x, float s, float inv) {
  float q = x * inv;
  q = fmaf(fmaf(-q, s, x), inv, q);                          // within a unit
  const float r = fmaf(-q, s, x);                            // what it leaves, exactly
  const int over = r != 0.f ? 1 : 0, away = (__float_as_int(r) ^ __float_as_int(q)) < 0 ? over : 0;
  return __int_as_float((__float_as_int(q) - away) | over);
}
__device__ __forceinline__ uint32_t fp8_two(float a, float b) {                    // a in the low byte
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t fp8_four_times(const float (&v)[4], float inv) {
  return fp8_two(v[0] * inv, v[1] * inv) | fp8_two(v[2] * inv, v[3] * inv) << 16;
}
// Where products with a little less and a little more than 1 / s give the same values, the quotients do too.
__device__ __forceinline__ uint32_t fp8_four(const float (&v)[4], float s) {
  const float inv = fp8_inverse(s);
  const uint32_t less = fp8_four_times(v, inv * (1.0f - 0x1p-21f)), more = fp8_four_times(v, inv * (1.0f + 0x1p-21f));
  if (less == more) return less;
  return fp8_two(fp8_quotient(v[0], s, inv), fp8_quotient(v[1], s, inv)) | fp8_two(fp8_quotient(v[2], s, inv), fp8_quotient(v[3], s, inv)) << 16;
}
__device__ __forceinline__ uint8_t fp8_one(float v, float s) {
  return __nv_cvt_float_to_fp8(fp8_quotient(v, s, fp8_inverse(s)), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint8_t fp8_one_times(float v, float inv) { return __nv_cvt_float_to_fp8(v * inv, __NV_SATFINITE, __NV_E4M3); }

}  // namespace atma
