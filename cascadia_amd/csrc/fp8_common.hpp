// fp8_common.hpp -- device helpers of the e4m3 kernels.
#pragma once
#include "int4_common.hpp"

namespace cai4 {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kFp8Least = 0x1p-96f;  // the least |max| of a group: 448 / it stays finite

// A group's divisor from its max|x|: x / (top / 448) is x * (hi + lo).  The two
// parts carry 448 / top to about 2^-48, so that q below is the quotient's own
// rounding: bf16 values often lie halfway between two codes, where a rounded
// 448 / top alone would choose by chance.
struct Fp8Div {
  float hi, lo, scale;
};
CAI4_DEV Fp8Div fp8_div(float top) {
  Fp8Div d;
  const float a = fmaxf(top, kFp8Least);
  d.hi = __fdiv_rn(kE4m3Max, a);
  // (an infinite maximum: codes and their products are NaN)
  d.lo = a <= 3.4028234e38f ? __fdiv_rn(__fmaf_rn(-d.hi, a, kE4m3Max), a) : 0.f;
  d.scale = __fdiv_rn(a, kE4m3Max);
  return d;
}
CAI4_DEV float fp8_quotient(const Fp8Div &d, float x) { return __fmaf_rn(x, d.hi, x * d.lo); }

// Four quotients (|q| <= 448, or NaN) as e4m3 codes, RNE.
CAI4_DEV uint32_t fp8_pack4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// Eight codes as bf16 (exact).
CAI4_DEV bf16x8_t fp8_to_bf16(uint32_t lo, uint32_t hi) {
  bf16x8_t r = {};
#ifdef __HIP_DEVICE_COMPILE__
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  r = bf16x8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
#endif
  return r;
}

// The products of a lane's 32 codes (k-slots shared by both operands) added to
// c, over bf16: exact products, f32 sums.
CAI4_DEV f32x4_t mfma_codes(const u32x4_t a[2], const u32x4_t b[2], f32x4_t c) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_to_bf16(a[h].x, a[h].y),
                                                fp8_to_bf16(b[h].x, b[h].y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_to_bf16(a[h].z, a[h].w),
                                                fp8_to_bf16(b[h].z, b[h].w), c, 0, 0, 0);
  }
  return c;
}

}  // namespace
}  // namespace cai4
