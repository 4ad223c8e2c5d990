// Block-scaled (MX) formats: 32 neighbours of a row share one scale, a power
// of two held as its biased exponent in a byte (e8m0; 255 is NaN).
//   MXFP8: e4m3 values, scale 2^e with the least e for which
//          max|x| <= 448 * 2^e, so that nothing saturates.
//   MXFP4: e2m1 values, two in a byte, the even k in the low half.
// A block that holds a NaN or an infinity is NaN throughout.
#pragma once
#include "fi/common.hpp"

namespace fi {

constexpr int kMxBlock = 32;

// The magnitude bits of a float order like the magnitudes, with every NaN
// above infinity: their unsigned maximum finds both, where fmaxf drops a NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

// Scale byte for a block whose largest magnitude has these bits. With
// max = m * 2^x, 1 <= m < 2, and 448 = 1.75 * 2^8 the exponent is x - 8, or
// one more where m > 1.75: whole-number work, so it is exact.
__device__ __forceinline__ uint32_t mxfp8_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  int byte = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u);
  return (uint32_t)(byte > 0 ? byte : 0);
}

// 2^-(byte - 127), exact for every byte that mxfp8_scale_byte returns for a
// finite block (0..247).
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}

// Eight scaled values as e4m3, rounded to nearest even. `bad` writes NaN.
__device__ __forceinline__ uint2 mxfp8_pack8(const float* y, float inv, bool bad) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
  return bad ? make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu) : make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Maximum over the four lanes of a quad (lanes 4i .. 4i + 3), in registers.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);
  v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);
  return v > o ? v : o;
}

// Maximum over a half of the wave (lanes 0 .. 31 or 32 .. 63).
__device__ __forceinline__ uint32_t max32(uint32_t v) {
#pragma unroll
  for (int i = 1; i < 32; i *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, i);
    v = v > o ? v : o;
  }
  return v;
}

}  // namespace fi
