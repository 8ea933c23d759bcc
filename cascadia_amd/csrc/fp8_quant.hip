// fp8_quant.hip -- values to e4m3 codes and f32 scales: rows in groups of 128
// columns (activations), or blocks of 128 x 128 (weights, at load).
//
// top = max(max|x|, 2^-96) over the group, scale = top / 448, code = e4m3(x /
// scale), to nearest even.  (Below 2^-96 codes shrink to zero rather than the
// divisor growing past f32.)  A group that holds an infinity gives NaN codes or
// an infinite scale, and so a NaN in every product with it.
//
// Bound: HBM, each value read and its code written once.  4096 x 7168 bf16 rows: 17
// us (5.2 TB/s, some of it from the Infinity Cache); 7104 x 8112 in blocks: 39 us (4.4
// TB/s; a copy reaches 4.87).
#include "fp8.hpp"
#include "fp8_common.hpp"
#include "fp8_quant.hpp"

namespace cai4 {
namespace {

template <bool F32>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const void *x, size_t groups, int K, int KB,
                                                       uint8_t *codes, float *scales, int ld) {
  quantize_rows_step<F32>(blockIdx.x, x, groups, K, KB, codes, scales, ld);
}

__global__ __launch_bounds__(256) void fp8_pad_kernel(const float *scales, size_t n, int KB,
                                                      float *to, int ld) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const size_t row = i / KB;
  to[row * ld + (i - row * KB)] = scales[i];
}

// A workgroup per block: 16 rows at a time, eight passes, held in registers.
__global__ __launch_bounds__(256) void fp8_blocks_kernel(const uint16_t *w, int N, int K, int KB,
                                                         uint8_t *codes, float *scales) {
  __shared__ float tops[4];
  const int nb = blockIdx.y, kb = blockIdx.x;
  const int col = kb * kFp8Block + 8 * (threadIdx.x & 15);
  const int row0 = nb * kFp8Block + (threadIdx.x >> 4);
  u32x4_t v[8];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = u32x4_t{0u, 0u, 0u, 0u};
    if (col < K && row0 + 16 * i < N)
      v[i] = *reinterpret_cast<const u32x4_t *>(w + (size_t)(row0 + 16 * i) * K + col);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, max_abs(v[i], false));
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const Fp8Div d = fp8_div(top);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col < K && row0 + 16 * i < N)
      *reinterpret_cast<u32x2_t *>(codes + (size_t)(row0 + 16 * i) * K + col) = codes_bf16(v[i], d);
  if (threadIdx.x == 0) scales[(size_t)nb * KB + kb] = d.scale;
}

// A workgroup per block: 16 bytes per thread, eight threads to a row, 32 rows at a time.
__global__ __launch_bounds__(256) void fp8_arrange_kernel(const uint8_t *codes, int N, int K, int NB,
                                                          int KB, uint8_t *tiled) {
  const size_t b = blockIdx.x, m = b / ((size_t)NB * KB);
  const int r = (int)(b - m * NB * KB), nb = r / KB, kb = r - nb * KB;
  const int row = threadIdx.x >> 3, at = (threadIdx.x & 7) * 16, col = kb * kFp8Block + at;
  uint8_t *to = tiled + b * kFp8BlockBytes + at;
  u32x4_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = nb * kFp8Block + row + 32 * i;
    v[i] = u32x4_t{0u, 0u, 0u, 0u};
    if (n < N && col < K)
      v[i] = *reinterpret_cast<const u32x4_t *>(codes + (m * N + n) * K + col);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4_t *>(to + (row + 32 * i) * 128) = v[i];
}

}  // namespace

hipError_t fp8_tile_weights(const uint8_t *codes, int count, int N, int K, uint8_t *tiled,
                            hipStream_t st) {
  const int NB = fp8_blocks(N), KB = fp8_blocks(K);
  const size_t blocks = (size_t)count * NB * KB;
  if (!launch_fits(blocks, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(fp8_arrange_kernel, dim3((unsigned)blocks), dim3(256), 0, st, codes, N, K, NB, KB,
                     tiled);
  return hipGetLastError();
}

hipError_t fp8_quantize_rows(const void *x, bool x_f32, size_t rows, int K, uint8_t *codes,
                             float *scales, int ld, hipStream_t st) {
  const int KB = fp8_blocks(K);
  const size_t groups = rows * KB;
  if (groups == 0) return hipSuccess;
  if (!launch_fits((groups + kRowGroups - 1) / kRowGroups, 256)) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((groups + kRowGroups - 1) / kRowGroups)), block(256);
  if (x_f32)
    hipLaunchKernelGGL(fp8_rows_kernel<true>, grid, block, 0, st, x, groups, K, KB, codes, scales,
                       ld);
  else
    hipLaunchKernelGGL(fp8_rows_kernel<false>, grid, block, 0, st, x, groups, K, KB, codes, scales,
                       ld);
  return hipGetLastError();
}

hipError_t fp8_pad_scales(const float *scales, size_t rows, int KB, float *to, int ld,
                          hipStream_t st) {
  const size_t n = rows * KB;
  if (!launch_fits((n + 255) / 256, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(fp8_pad_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, scales, n,
                     KB, to, ld);
  return hipGetLastError();
}

hipError_t fp8_quantize_blocks(const uint16_t *w, int N, int K, uint8_t *codes, float *scales,
                               hipStream_t st) {
  const int KB = fp8_blocks(K);
  hipLaunchKernelGGL(fp8_blocks_kernel, dim3(KB, fp8_blocks(N)), dim3(256), 0, st, w, N, K, KB,
                     codes, scales);
  return hipGetLastError();
}

}  // namespace cai4
