// fp8_gemm.hip -- matrix product of e4m3 codes with a scale per block of 128.
//
//   y[t, n] = sum_kb xs[t, kb] ws[n / 128, kb] sum_{k in kb} x[t, k] w[n, k]
//
// Weight rows are the A operand of 16x16 MFMAs, tokens the B operand, so that a
// lane's results are four neighbouring outputs of one token and need one scale.
// A block's partial sum starts from zero and enters the f32 sum with the two
// scales' product.  Which of a block's columns sits in which k-slot does not
// matter as long as both operands agree: a lane takes bytes 16 c ... and 64 + 16
// c ... of its row's 128 (c = lane >> 4), so that one load instruction reads 64
// neighbouring bytes of each of 16 rows.
//
// The 8-bit MFMAs do not add in f32: measured against 64 bits, the sum of a
// block's 128 products is 1.5e-5 off (normal values; 5e-5 for codes spread over
// all exponents), in every form of the instruction, where the same codes as bf16
// (exact) give 1e-8.  So the products run on the bf16 MFMAs, codes converted in
// registers.
#include "fp8.hpp"
#include "fp8_common.hpp"
#include "fp8_rows.hpp"
#include "lds_dma.hpp"

namespace cai4 {
namespace {

// 16 bytes at byte `off` (zeros past the range).
CAI4_DEV u32x4_t load16(rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

// ---------------------------------------------------------------------------
// few rows: weights from HBM straight into registers
// ---------------------------------------------------------------------------

// A workgroup: 16 weight rows (SW: the same 16 of gate and up), 16 tokens, its
// waves taking the k-blocks in turn and adding up through LDS in wave order.
constexpr int kFewWaves = 8;

template <bool SW>
__global__ __launch_bounds__(64 * kFewWaves) void fp8_few_kernel(Fp8Gemm g) {
  constexpr int W = kFewWaves, MT = SW ? 2 : 1;
  __shared__ f32x4_t part[W][MT][64];
  const int lane = threadIdx.x & 63, l15 = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ntiles = (g.N + 15) >> 4, mt = blockIdx.x / ntiles;
  if (g.chunks && mt >= *g.n_chunks) return;  // the whole workgroup
  const Rows rows = rows_of(g, mt, 16);
  const int n0 = (blockIdx.x - mt * ntiles) * 16, KB = (g.K + 127) >> 7, NB = (g.N + 127) >> 7;
  const int nr = g.N - n0 < 16 ? g.N - n0 : 16;
  const uint8_t *w = g.w + (size_t)rows.expert * g.w_stride + (size_t)n0 * g.K;
  const float *ws = g.ws + (size_t)rows.expert * g.ws_stride + (size_t)(n0 >> 7) * KB;
  const rsrc_t wr0 = rsrc(w, (size_t)nr * g.K);
  const rsrc_t wr1 = rsrc(SW ? w + (size_t)g.N * g.K : w, (size_t)nr * g.K);
  const bool tok = l15 < rows.count;
  const int grow = rows.row0 + (tok ? l15 : 0);
  const int xrow = g.row_map ? g.row_map[grow] : grow;
  const uint8_t *x = g.x + (size_t)xrow * g.K;
  const float *xs = g.xs + (size_t)xrow * g.ld_xs;
  f32x4_t acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < KB; kb += W) {
    const int c0 = kb * 128 + 16 * c, c1 = c0 + 64;
    const uint32_t o0 = l15 < nr && c0 < g.K ? (uint32_t)(l15 * g.K + c0) : kDmaOOB;
    const uint32_t o1 = l15 < nr && c1 < g.K ? (uint32_t)(l15 * g.K + c1) : kDmaOOB;
    u32x4_t a[MT][2], b[2];
    a[0][0] = load16(wr0, o0);
    a[0][1] = load16(wr0, o1);
    if (SW) {
      a[MT - 1][0] = load16(wr1, o0);
      a[MT - 1][1] = load16(wr1, o1);
    }
    b[0] = b[1] = u32x4_t{0u, 0u, 0u, 0u};
    if (tok && c0 < g.K) b[0] = *reinterpret_cast<const u32x4_t *>(x + c0);
    if (tok && c1 < g.K) b[1] = *reinterpret_cast<const u32x4_t *>(x + c1);
    const float s = tok ? xs[kb] : 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const f32x4_t p = mfma_codes(a[m], b, f32x4_t{0.f, 0.f, 0.f, 0.f});
      const float sw = s * ws[(size_t)m * NB * KB + kb];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] = __fmaf_rn(p[i], sw, acc[m][i]);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) part[wave][m][lane] = acc[m];
  __syncthreads();
  if (wave > 0) return;
  f32x4_t v[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    v[m] = part[0][m][lane];
    for (int q = 1; q < W; ++q) v[m] += part[q][m][lane];
  }
  if (SW) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[0][i] = silu_f32(v[0][i]) * v[MT - 1][i];
  }
  if (tok) store4(g, (size_t)grow, n0 + 4 * c, v[0]);
}

}  // namespace

bool fp8_tiles(int M, int N, int K) { return M > 64; }

hipError_t fp8_gemm(const Fp8Gemm &g, hipStream_t st) {
  if (g.chunks ? g.chunk_rows > 16 : fp8_tiles(g.M, g.N, g.K)) return fp8_tile_gemm(g, st);
  const size_t tiles = (size_t)((g.N + 15) / 16) * (g.chunks ? g.max_chunks : (g.M + 15) / 16);
  if (tiles > 0x7FFFFFFFu) return hipErrorInvalidValue;
  const dim3 grid((unsigned)tiles);
  if (g.swiglu)
    hipLaunchKernelGGL(fp8_few_kernel<true>, grid, dim3(64 * kFewWaves), 0, st, g);
  else
    hipLaunchKernelGGL(fp8_few_kernel<false>, grid, dim3(64 * kFewWaves), 0, st, g);
  return hipGetLastError();
}

}  // namespace cai4
