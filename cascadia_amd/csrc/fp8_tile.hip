// fp8_tile.hip -- products of many rows of e4m3 codes: tiles of up to 256
// weight rows x 256 tokens staged through LDS, for one matrix or for the row
// groups of many experts in one launch.
//
// A block of 128 columns is one step: both operands' codes go global -> LDS by
// loads with an LDS destination (two stages), each wave reads the fragments of
// its 16 NI weight rows and 16 NJ tokens, and every 16 x 16 tile's partial sum
// over the block (starting from zero) enters its f32 sum with the product of the
// two scales: one f32 scale per token and block, since a wave's weight rows lie
// in one block of 128.
//
// Two forms of the products:
//   fast   one 16x16x128 8-bit MFMA per tile and block.  It adds groups of eight
//          products aligned to the largest, whose bits below 2^-14 of it are
//          dropped: about 1.5e-5 of the result, where rounding an output to bf16
//          takes 2e-3.  Used where the output is bf16.
//   exact  the codes converted to bf16 in registers (exact) and four 16x16x32
//          MFMAs: f32 sums, at half the rate.  Used for f32 outputs, and for
//          SwiGLU, whose result is quantised again: 1.5e-5 there moves 1 value
//          in 3,000 to the neighbouring code.
//
// LDS: a row of 128 bytes is eight 16-byte chunks, chunk c of row r in slot
// c ^ (r / 2 & 7), so that the 16 rows that a fragment read touches at once lie
// in different banks.  A lane takes chunks c and c + 4 (c = lane >> 4) of its
// row for both operands.
//
// Order: weight tiles outside, tokens inside.  The tokens' fragments stay in
// registers for the block, the weights' are read one tile ahead.  Before the
// last weight tile nothing of the stage is left to read: there the one barrier
// of the block stands, which also publishes the next stage; its loads were
// issued one block earlier, those of the stage after it go into the freed one.
#include "fp8.hpp"
#include "fp8_common.hpp"
#include "fp8_rows.hpp"
#include "lds_dma.hpp"

namespace cai4 {
namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

CAI4_DEV f32x4_t mfma_fp8(const u32x4_t a[2], const u32x4_t b[2]) {
  f32x4_t p = {0.f, 0.f, 0.f, 0.f};
#ifdef __HIP_DEVICE_COMPILE__
  const i32x8_t x = {(int)a[0].x, (int)a[0].y, (int)a[0].z, (int)a[0].w,
                     (int)a[1].x, (int)a[1].y, (int)a[1].z, (int)a[1].w};
  const i32x8_t y = {(int)b[0].x, (int)b[0].y, (int)b[0].z, (int)b[0].w,
                     (int)b[1].x, (int)b[1].y, (int)b[1].z, (int)b[1].w};
  // formats 0, 0: e4m3 both; no block scales
  p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, p, 0, 0, 0, 0, 0, 0);
#endif
  return p;
}

// Keeps these values' computation where it is written: between scheduling
// barriers arithmetic whose result nothing there uses is moved to the end.
CAI4_DEV void pin(f32x4_t &v) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(v));
#endif
}

// WN x WM waves of 16 NI weight rows x 16 NJ tokens.  SW: a wave's first NI / 2
// tiles are gate rows, the others the same rows of up.
template <int NI, int NJ, int WN, int WM, bool SW>
struct Tile {
  static constexpr int W = WN * WM, BN = 16 * NI * WN, BM = 16 * NJ * WM;
  static constexpr int OUT = SW ? BN / 2 : BN;  // output columns
  static constexpr int STAGE = (BN + BM) * 128;
  static constexpr int PW = BN / 8 / W, PX = BM / 8 / W;  // 1 KB loads per wave and stage
  static_assert(PW * W * 8 == BN && PX * W * 8 == BM, "pieces");
  static_assert(128 % (16 * NI / (SW ? 2 : 1)) == 0, "a wave's rows lie in one scale block");
  static_assert(2 * STAGE <= 160 * 1024, "LDS");
};

template <int NI, int NJ, int WN, int WM, bool SW, bool EXACT>
__global__ __launch_bounds__(64 * WN * WM) void fp8_tile_kernel(Fp8Gemm g, int ntiles) {
  using P = Tile<NI, NJ, WN, WM, SW>;
  __shared__ __attribute__((aligned(1024))) uint8_t st[2 * P::STAGE];
  const int lane = threadIdx.x & 63, l15 = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int mt = blockIdx.x / ntiles, n0 = (blockIdx.x - mt * ntiles) * P::OUT;
  const Rows rows = rows_of(g, mt, P::BM);
  if (rows.count <= 0) return;  // the whole workgroup
  const int KB = (g.K + 127) >> 7, NB = (g.N + 127) >> 7;
  const int nr = g.N - n0 < P::OUT ? g.N - n0 : P::OUT;
  // this wave loads rows of the weights (SwiGLU: the first half gate, the others up)
  const uint8_t *w = g.w + (size_t)rows.expert * g.w_stride + (size_t)n0 * g.K +
                     (SW && wave >= P::W / 2 ? (size_t)g.N * g.K : 0);
  const rsrc_t wr = rsrc_scalar(w, (size_t)nr * g.K);
  const rsrc_t xr = g.row_map ? rsrc_scalar(g.x, (size_t)g.x_rows * g.K)
                              : rsrc_scalar(g.x + (size_t)rows.row0 * g.K,
                                            (size_t)rows.count * g.K);
  const rsrc_t sr = g.row_map ? rsrc_scalar(g.xs, (size_t)g.x_rows * KB * 4)
                              : rsrc_scalar(g.xs + (size_t)rows.row0 * KB,
                                            (size_t)rows.count * KB * 4);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const lds_void *)st);

  // ---- this wave's loads of a stage: 1 KB pieces of eight rows, PW of the
  // weights and PX of the tokens; lane i loads the chunk that belongs in slot i & 7
  // of row i >> 3 ----
  uint32_t vw[P::PW], vx[P::PX];
  auto chunk_of = [&](int row) { return (lane & 7) ^ ((row >> 1) & 7); };
#pragma unroll
  for (int q = 0; q < P::PW; ++q) {
    const int row = (wave * P::PW + q) * 8 + (lane >> 3), r = SW ? row & (P::BN / 2 - 1) : row;
    vw[q] = r < nr ? (uint32_t)(r * g.K) + 16 * chunk_of(row) : kDmaOOB;
  }
#pragma unroll
  for (int q = 0; q < P::PX; ++q) {
    const int r = (wave * P::PX + q) * 8 + (lane >> 3);
    vx[q] = r >= rows.count ? kDmaOOB
            : (g.row_map ? (uint32_t)g.row_map[rows.row0 + r] * (uint32_t)g.K
                         : (uint32_t)(r * g.K)) + 16 * chunk_of(r);
  }
  auto issue = [&](int kb) {
    const uint32_t to = lds0 + (kb & 1) * P::STAGE, soff = (uint32_t)kb * 128;
    const int left = g.K - 128 * kb;  // a short last block reads zeros past it
#pragma unroll
    for (int q = 0; q < P::PW; ++q) {
      const int piece = wave * P::PW + q;
      const uint32_t v = 16 * chunk_of(piece * 8 + (lane >> 3)) < left ? vw[q] : kDmaOOB;
      lds_dma<16>(wr, to + piece * 1024, v, soff);
    }
#pragma unroll
    for (int q = 0; q < P::PX; ++q) {
      const int piece = wave * P::PX + q;
      const uint32_t v = 16 * chunk_of(piece * 8 + (lane >> 3)) < left ? vx[q] : kDmaOOB;
      lds_dma<16>(xr, to + P::BN * 128 + piece * 1024, v, soff);
    }
  };

  // ---- scales: one per token and block, times the weight rows' ----
  uint32_t so[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = (wm * NJ + j) * 16 + l15;
    so[j] = r >= rows.count ? kDmaOOB
            : g.row_map     ? (uint32_t)g.row_map[rows.row0 + r] * (uint32_t)KB * 4
                            : (uint32_t)(r * KB) * 4;
  }
  const int nw = SW ? n0 + wn * 8 * NI : n0 + wn * 16 * NI;  // this wave's first row
  const bool idle = nw >= g.N;
  const size_t eo = (size_t)rows.expert * g.ws_stride;
  const float *ws = g.ws + eo + (size_t)((idle ? n0 : nw) >> 7) * KB;
  constexpr int NS = SW ? 2 : 1;
  float xv[NJ], wv[NS], s[NS][NJ];
  auto load_scales = [&](int kb) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      xv[j] = bitsf(__builtin_amdgcn_raw_buffer_load_b32(sr, so[j], kb * 4, 0));
    wv[0] = ws[kb];
    if (SW) wv[NS - 1] = ws[(size_t)NB * KB + kb];
  };
  auto take_scales = [&](float (&to)[NS][NJ]) {
#pragma unroll
    for (int m = 0; m < NS; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j) to[m][j] = xv[j] * wv[m];
  };

  // ---- fragments: chunks c and c + 4 of rows 16 i + l15 ----
  const uint32_t fo = lds0 + l15 * 128 + ((c ^ ((l15 >> 1) & 7)) << 4);
  const uint32_t fw = fo + (SW ? wn * NI * 8 : wn * NI * 16) * 128;
  const uint32_t fx = fo + (P::BN + wm * NJ * 16) * 128;
  u32x4_t a[2][2], b[NJ][2];
  auto read_a = [&](uint32_t base, int i, int to) {
    const int row = SW && i >= NI / 2 ? P::BN / 2 + 16 * (i - NI / 2) : 16 * i;
    a[to][0] = lds_at<u32x4_t>(base + fw, row * 128);
    a[to][1] = lds_at<u32x4_t>((base + fw) ^ 64, row * 128);
  };
  auto read_b = [&](uint32_t base, int j) {
    b[j][0] = lds_at<u32x4_t>(base + fx, j * 2048);
    b[j][1] = lds_at<u32x4_t>((base + fx) ^ 64, j * 2048);
  };

  f32x4_t acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  load_scales(0);
  issue(0);
  dma_wait_barrier<0>();
  take_scales(s);
  if (KB > 1) issue(1);
#pragma unroll
  for (int j = 0; j < NJ; ++j) read_b(0, j);
  read_a(0, 0, 0);
  constexpr int LAG = 2;  // MFMAs between one and the use of its result
  f32x4_t p[LAG + 1];
  for (int kb = 0; kb < KB; ++kb) {
    const uint32_t base = (kb & 1) * P::STAGE, next = P::STAGE - base;
    load_scales(kb + 1 < KB ? kb + 1 : kb);
    float sn[NS][NJ];
    auto add = [&](int slot) {
      const int i = slot / NJ, j = slot % NJ;
      const float f = s[SW && i >= NI / 2][j];
#pragma unroll
      for (int v = 0; v < 4; ++v)
        acc[i][j][v] = __fmaf_rn(p[slot % (LAG + 1)][v], f, acc[i][j][v]);
      pin(acc[i][j]);
    };
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (i + 1 < NI) {
        read_a(base, i + 1, (i + 1) & 1);
      } else {
        dma_wait_barrier<0>();
        take_scales(sn);
        if (kb + 2 < KB) issue(kb + 2);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int slot = i * NJ + j;
        if constexpr (EXACT)
          p[slot % (LAG + 1)] = mfma_codes(a[i & 1], b[j], f32x4_t{0.f, 0.f, 0.f, 0.f});
        else
          p[slot % (LAG + 1)] = mfma_fp8(a[i & 1], b[j]);
        if (slot >= LAG) add(slot - LAG);
        if (i + 1 == NI) read_b(next, j);  // (past the last block: not used)
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    read_a(next, 0, 0);
#pragma unroll
    for (int q = LAG; q > 0; --q) add(NI * NJ - q);
#pragma unroll
    for (int m = 0; m < NS; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j) s[m][j] = sn[m][j];
  }

  if (idle) return;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = (wm * NJ + j) * 16 + l15;
    if (r >= rows.count) continue;
    const size_t row = (size_t)rows.row0 + r;
    if constexpr (SW) {
#pragma unroll
      for (int i = 0; i < NI / 2; ++i) {
        f32x4_t h;
#pragma unroll
        for (int v = 0; v < 4; ++v) h[v] = silu_f32(acc[i][j][v]) * acc[i + NI / 2][j][v];
        store4(g, row, nw + 16 * i + 4 * c, h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) store4(g, row, nw + 16 * i + 4 * c, acc[i][j]);
    }
  }
}

template <int NI, int NJ, int WN, int WM, bool SW, bool EXACT>
hipError_t launch(const Fp8Gemm &g, hipStream_t st) {
  using P = Tile<NI, NJ, WN, WM, SW>;
  const int nt = (g.N + P::OUT - 1) / P::OUT;
  const size_t tiles = (size_t)nt * (g.chunks ? g.max_chunks : (g.M + P::BM - 1) / P::BM);
  if (tiles > 0x7FFFFFFFu) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fp8_tile_kernel<NI, NJ, WN, WM, SW, EXACT>), dim3((unsigned)tiles),
                     dim3(64 * P::W), 0, st, g, nt);
  return hipGetLastError();
}

}  // namespace

hipError_t fp8_tile_gemm(const Fp8Gemm &g, hipStream_t st) {
  if (g.swiglu) return launch<8, 2, 2, 4, true, true>(g, st);
  if (g.out_f32) return launch<8, 2, 2, 4, false, true>(g, st);
  if (g.chunks) return launch<8, 2, 2, 4, false, false>(g, st);
  return launch<8, 4, 2, 4, false, false>(g, st);
}

}  // namespace cai4
