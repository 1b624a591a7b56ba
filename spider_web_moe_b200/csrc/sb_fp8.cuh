// Block-scaled e4m3: the scale of a block and the rounding of its values,
// shared by the quantisation kernels and the products' quantised epilogues.
#pragma once
#include "sb_common.cuh"

namespace sb {

// |v| as an integer that orders like |v|, with NaN above inf.
SB_DEVINL uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Fp8Scale {
  float scale;  // a / 448
  float inv;    // 448 / a
};

// a = max(amax, 2^-100) from the amax's bits (an integer maximum, so NaN stays);
// both divisions round to nearest.
SB_DEVINL Fp8Scale fp8_scale(uint32_t amax_bits) {
  const float a = __uint_as_float(max(amax_bits, __float_as_uint(0x1p-100f)));
  return {__fdiv_rn(a, 448.f), __fdiv_rn(448.f, a)};
}

// Four values to e4m3 (round to nearest even, saturating; NaN stays NaN).
SB_DEVINL uint32_t fp8_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Four bf16 values (two per word) times inv, to e4m3.
SB_DEVINL uint32_t fp8_pack4_bf16(uint32_t a, uint32_t b, float inv) {
  return fp8_pack4(__uint_as_float(a << 16) * inv, __uint_as_float(a & 0xffff0000u) * inv, __uint_as_float(b << 16) * inv,
                   __uint_as_float(b & 0xffff0000u) * inv);
}

}  // namespace sb
