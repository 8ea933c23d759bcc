// fp8_rows.hpp -- what the kernels of fp8_gemm.hip and fp8_tile.hip share: a
// workgroup's rows, and the store of its outputs.
#pragma once
#include "fp8.hpp"
#include "int4_common.hpp"

namespace cai4 {
namespace {

// The rows of one workgroup: of the whole matrix, or of one chunk.
struct Rows {
  int expert, row0, count;
};
CAI4_DEV Rows rows_of(const Fp8Gemm &g, int chunk, int per) {
  Rows r;
  if (g.chunks) {
    const Fp8Chunk c = g.chunks[chunk];
    r.expert = __builtin_amdgcn_readfirstlane(c.expert);
    r.row0 = __builtin_amdgcn_readfirstlane(c.row0);
    r.count = __builtin_amdgcn_readfirstlane(c.count);
  } else {
    r.expert = 0;
    r.row0 = chunk * per;
    r.count = g.M - r.row0 < per ? g.M - r.row0 : per;
  }
  return r;
}

// Four neighbouring outputs n .. n + 3 of one token.
CAI4_DEV void store4(const Fp8Gemm &g, size_t row, int n, f32x4_t v) {
  const size_t at = row * g.N + n;
  if (g.out_f32) {
    float *y = static_cast<float *>(g.y) + at;
    if (n + 4 <= g.N && ((uintptr_t)y & 15) == 0) {
      *reinterpret_cast<f32x4_t *>(y) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < g.N) y[i] = v[i];
    }
  } else {
    uint16_t *y = static_cast<uint16_t *>(g.y) + at;
    u32x2_t b;
    b.x = f32_to_bf16_rne(v.x) | (f32_to_bf16_rne(v.y) << 16);
    b.y = f32_to_bf16_rne(v.z) | (f32_to_bf16_rne(v.w) << 16);
    if (n + 4 <= g.N && ((uintptr_t)y & 7) == 0) {
      *reinterpret_cast<u32x2_t *>(y) = b;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < g.N) y[i] = (uint16_t)(b[i >> 1] >> (16 * (i & 1)));
    }
  }
}

}  // namespace
}  // namespace cai4
