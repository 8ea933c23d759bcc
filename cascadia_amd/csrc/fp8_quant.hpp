// fp8_quant.hpp -- device code of the quantisation of rows (fp8_quant.hip,
// fp8_moe.hip).
#pragma once
#include "fp8.hpp"
#include "fp8_common.hpp"

namespace cai4 {
namespace {

CAI4_DEV float max_abs(u32x4_t v, bool f32) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (f32) {
      m = fmaxf(m, fabsf(bitsf(v[e])));
    } else {
      m = fmaxf(m, fabsf(bitsf(v[e] << 16)));
      m = fmaxf(m, fabsf(bitsf(v[e] & 0xFFFF0000u)));
    }
  }
  return m;
}

// Eight bf16 values as codes.
CAI4_DEV u32x2_t codes_bf16(u32x4_t v, const Fp8Div &d) {
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    q[e] = fp8_quotient(d, bitsf((e & 1) ? v[e >> 1] & 0xFFFF0000u : v[e >> 1] << 16));
  return u32x2_t{fp8_pack4(q[0], q[1], q[2], q[3]), fp8_pack4(q[4], q[5], q[6], q[7])};
}
CAI4_DEV u32x2_t codes_f32(u32x4_t v, u32x4_t w, const Fp8Div &d) {
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = fp8_quotient(d, bitsf(e < 4 ? v[e & 3] : w[e & 3]));
  return u32x2_t{fp8_pack4(q[0], q[1], q[2], q[3]), fp8_pack4(q[4], q[5], q[6], q[7])};
}

// Sixteen lanes share a group, eight columns each.
constexpr int kRowGroups = 16;  // groups per workgroup of 256 threads
template <bool F32>
CAI4_DEV void quantize_rows_step(size_t block, const void *x, size_t groups, int K, int KB,
                                 uint8_t *codes, float *scales, int ld) {
  const size_t g = block * kRowGroups + (threadIdx.x >> 4);
  if (g >= groups) return;  // whole groups of 16 lanes
  const size_t row = g / KB;
  const int kb = (int)(g - row * KB), col = kb * kFp8Block + 8 * (threadIdx.x & 15);
  const bool in = col < K;  // (K is a multiple of 16)
  const size_t at = row * K + col;
  u32x4_t v = {0u, 0u, 0u, 0u}, w = v;
  if (in) {
    if (F32) {
      const float *f = static_cast<const float *>(x) + at;
      v = *reinterpret_cast<const u32x4_t *>(f);
      w = *reinterpret_cast<const u32x4_t *>(f + 4);
    } else {
      v = *reinterpret_cast<const u32x4_t *>(static_cast<const uint16_t *>(x) + at);
    }
  }
  float top = max_abs(v, F32);
  if (F32) top = fmaxf(top, max_abs(w, true));
#pragma unroll
  for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  const Fp8Div d = fp8_div(top);
  if (in)
    *reinterpret_cast<u32x2_t *>(codes + at) = F32 ? codes_f32(v, w, d) : codes_bf16(v, d);
  if ((threadIdx.x & 15) == 0) scales[row * ld + kb] = d.scale;
}

}  // namespace
}  // namespace cai4
