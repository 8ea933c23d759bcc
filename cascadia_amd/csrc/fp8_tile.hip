// fp8_tile.hip -- products of many rows of e4m3 codes: tiles of up to 256
// weight rows x 256 tokens staged through LDS, for one matrix or for the row
// groups of many experts in one launch.
//
// A block of 128 columns is one step: both operands' codes go global -> LDS by
// loads with an LDS destination (S stages), each wave reads the fragments of
// its 16 NI weight rows and 16 NJ tokens, and every 16 x 16 tile's partial sum
// over the block (starting from zero) enters its f32 sum with the product of the
// two scales: one f32 scale per token and block, since a wave's weight rows lie
// in one block of 128.
//
// Two forms of the products:
//   fast   one 16x16x128 8-bit MFMA per tile and block.  It adds groups of eight
//          products aligned to the largest, whose bits below 2^-13 of it are
//          dropped: about 1.5e-5 of the products' root sum of squares, where
//          rounding an output to bf16 takes 2e-3.  Used where the output is bf16.
//   exact  the codes converted to bf16 in registers (exact) and four 16x16x32
//          MFMAs: f32 sums, at half the rate.  Used for f32 outputs.
// A layer takes the form of its output for all its products.  SwiGLU's result is
// quantised to 4 bits of precision right here, where 1.5e-5 moves one value in some
// 3,000 to the neighbouring code.  2,048 tokens over 128 experts of 4096 x 1536, off
// the 64-bit output (relative, as a whole) and time: bf16 out 1.75e-3 (rounding it
// alone 1.66e-3), 795 us; f32 out 2.1e-4, 1100 us (with 8-bit sums 5.5e-4, 795).
//
// LDS: a row of 128 bytes is eight 16-byte chunks, chunk c of row r in slot
// c ^ (r / 2 & 7), so that the 16 rows that a fragment read touches at once lie
// in different banks.  A lane takes chunks c and c + 4 (c = lane >> 4) of its
// row for both operands.
//
// Order: weight tiles outside, tokens inside.  The tokens' fragments stay in
// registers for the block, the weights' are read one tile ahead.  Before the
// last weight tile nothing of the stage is left to read: there the one barrier
// of the block stands, which also publishes the next stage.  The freed one takes
// the loads of the block S further during the next block, one or two a pass
// (past the last block: loads out of range, so that every wait counts the same
// number).  Issued all at once behind the barrier they hold up every wave while the
// address unit works through them.
//
// What bounds it: a CU keeps some 64 cache lines in flight to its L2, about 14
// bytes a cycle at 390 cycles each, so requests count.  The tokens' scales, rows
// padded to 16 bytes, are read four blocks at a time; one by one they were a third
// of all requests.  Measured, M x N x K 4096 x 14336 x 4096, bf16 out: 251 us, 1.92
// PFLOP/s (one large library product of codes under one scale: 2.65 PFLOP/s); f32 out
// 427 us, 1.13 PFLOP/s.  Of 2,048 tokens over 128 experts of 4096 x 1536: gate and up
// 442 to 496 us, down 268 to 302.
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
template <int NI, int NJ, int WN, int WM, bool SW, int S>
struct Tile {
  static constexpr int W = WN * WM, BN = 16 * NI * WN, BM = 16 * NJ * WM;
  static constexpr int OUT = SW ? BN / 2 : BN;  // output columns
  static constexpr int STAGE = (BN + BM) * 128, WINDOW = BM * 16;  // codes; scales of four blocks
  static constexpr int SL = 16 * NJ / WN;  // tokens whose scales a wave loads
  static constexpr int XS = S * STAGE, NONE = XS + 2 * WINDOW, BYTES = NONE + SL * 16;
  static constexpr int PW = BN / 8 / W, PX = BM / 8 / W;  // 1 KB loads per wave and stage
  static_assert(PW * W * 8 == BN && PX * W * 8 == BM, "pieces");
  static_assert(128 % (16 * NI / (SW ? 2 : 1)) == 0, "a wave's rows lie in one scale block");
  static constexpr int LOADS = PW + PX + 1;
  static_assert(S >= 2 && S <= 4 && BYTES + (SW ? WN * BM * 4 : 0) <= 160 * 1024, "LDS");
  static_assert(SL * WN == 16 * NJ && SL <= 64, "a wave's scales are one load");
};

// A workgroup's place: m tile (or chunk) and n tile.  Workgroups go round the
// eight XCDs; each takes a run of neighbouring tiles, so that those that run
// together share rows of both operands in its L2.  One matrix: groups of 4 m
// tiles, n outside, m inside (32 workgroups: 4 x 8 tiles).  Experts, one after
// the other: n outside, the expert's chunks inside.
struct Place {
  int m, n;
};
CAI4_DEV Place place_of(const Fp8Gemm &g, int id, int mtiles, int ntiles) {
  const int total = mtiles * ntiles, per = (total + 7) >> 3, t = (id & 7) * per + (id >> 3);
  if ((id >> 3) >= per || t >= total) return Place{-1, 0};
  if (g.chunks) {
    const Fp8Chunk c = g.chunks[t / ntiles];  // some chunk of the tile's expert
    const int r = t - c.first * ntiles;
    return Place{__builtin_amdgcn_readfirstlane(c.first + r % c.number),
                 __builtin_amdgcn_readfirstlane(r / c.number)};
  }
  const int group = t / (4 * ntiles), r = t - group * 4 * ntiles;
  const int gm = mtiles - group * 4 < 4 ? mtiles - group * 4 : 4;
  return Place{group * 4 + r % gm, r / gm};
}

template <int NI, int NJ, int WN, int WM, bool SW, bool EXACT, int S>
__global__ __launch_bounds__(64 * WN * WM) void fp8_tile_kernel(Fp8Gemm g, int n_first, int ntiles) {
  using P = Tile<NI, NJ, WN, WM, SW, S>;
  __shared__ __attribute__((aligned(1024))) uint8_t st[P::BYTES];
  __shared__ float tops[SW ? WN : 1][SW ? P::BM : 1];
  const int lane = threadIdx.x & 63, l15 = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int mtiles = g.chunks ? __builtin_amdgcn_readfirstlane(*g.n_chunks)
                              : (g.M + P::BM - 1) / P::BM;
  const Place at = place_of(g, blockIdx.x, mtiles, ntiles);
  if (at.m < 0) return;  // the whole workgroup
  const int n0 = n_first + at.n * P::OUT;
  const Rows rows = rows_of(g, at.m, P::BM);
  const int KB = (g.K + 127) >> 7, NB = (g.N + 127) >> 7;
  // this workgroup's blocks: all, or slice blockIdx.y of g.kper (a multiple of 4)
  const int first = g.kper ? (int)blockIdx.y * g.kper : 0;
  const int end = g.kper && first + g.kper < KB ? first + g.kper : KB;
  const int cols = end * 128 < g.K ? end * 128 : g.K;
  const int nr = g.N - n0 < P::OUT ? g.N - n0 : P::OUT;
  // this wave loads rows of the weights (SwiGLU: the first half gate, the others up)
  const uint32_t band = (uint32_t)(KB * kFp8BlockBytes);  // 128 rows, in blocks
  const size_t matrix = g.w_tiled ? (size_t)NB * band : (size_t)g.N * g.K;
  const uint8_t *w = g.w + (size_t)rows.expert * g.w_stride +
                     (g.w_tiled ? (size_t)(n0 >> 7) * band : (size_t)n0 * g.K) +
                     (SW && wave >= P::W / 2 ? matrix : 0);
  const rsrc_t wr = rsrc_scalar(w, g.w_tiled ? (size_t)((nr + 127) >> 7) * band
                                             : (size_t)nr * g.K);
  const uint32_t wstep = g.w_tiled ? (uint32_t)kFp8BlockBytes : 128u;  // per block of K
  const rsrc_t xr = g.row_map ? rsrc_scalar(g.x, (size_t)g.x_rows * g.K)
                              : rsrc_scalar(g.x + (size_t)rows.row0 * g.K,
                                            (size_t)rows.count * g.K);
  const rsrc_t sr = g.row_map ? rsrc_scalar(g.xs, (size_t)g.x_rows * g.ld_xs * 4)
                              : rsrc_scalar(g.xs + (size_t)rows.row0 * g.ld_xs,
                                            (size_t)rows.count * g.ld_xs * 4);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const lds_void *)st);

  // ---- this wave's loads of a stage: 1 KB pieces of eight rows, PW of the
  // weights and PX of the tokens; lane i loads the chunk that belongs in slot i & 7
  // of row i >> 3 ----
  uint32_t vw[P::PW], vx[P::PX];
  auto chunk_of = [&](int row) { return (lane & 7) ^ ((row >> 1) & 7); };
#pragma unroll
  for (int q = 0; q < P::PW; ++q) {
    const int row = (wave * P::PW + q) * 8 + (lane >> 3), r = SW ? row & (P::BN / 2 - 1) : row;
    const uint32_t at = g.w_tiled ? (uint32_t)(r >> 7) * band + (uint32_t)(r & 127) * 128
                                  : (uint32_t)(r * g.K);
    vw[q] = r < nr ? at + 16 * chunk_of(row) : kDmaOOB;
  }
#pragma unroll
  for (int q = 0; q < P::PX; ++q) {
    const int r = (wave * P::PX + q) * 8 + (lane >> 3);
    vx[q] = r >= rows.count ? kDmaOOB
            : (g.row_map ? (uint32_t)g.row_map[rows.row0 + r] * (uint32_t)g.K
                         : (uint32_t)(r * g.K)) + 16 * chunk_of(r);
  }
  // scales: 16 bytes, four blocks' of a token, with every fourth stage (two windows)
  uint32_t vs = kDmaOOB;
  const int s0 = wm * NJ * 16 + wn * P::SL;
  if (s0 + lane < rows.count)
    vs = (g.row_map && lane < P::SL ? (uint32_t)g.row_map[rows.row0 + s0 + lane]
                                    : (uint32_t)(s0 + lane)) * (uint32_t)g.ld_xs * 4;
  // load q of this wave for block kb into the stage at `to`.  A short last block
  // reads zeros past its end: chunks of pieces of one parity are cut alike.
  auto cut = [&](int kb, int parity) {
    return 16 * (((lane & 7) ^ ((4 * parity + (lane >> 4)) & 7))) < cols - 128 * kb;
  };
  auto load1 = [&](int q, int kb, uint32_t to, bool even, bool odd) {
    if (q < P::PW) {
      const int piece = wave * P::PW + q;
      lds_dma<16>(wr, to + piece * 1024, (piece & 1 ? odd : even) ? vw[q] : kDmaOOB,
                  (uint32_t)kb * wstep);
    } else if (q < P::PW + P::PX) {
      const int piece = wave * P::PX + q - P::PW;
      lds_dma<16>(xr, to + P::BN * 128 + piece * 1024,
                  (piece & 1 ? odd : even) ? vx[q - P::PW] : kDmaOOB, (uint32_t)kb * 128);
    } else {
      // (in the other stages, and past the end, zeros to a place that nothing reads)
      const bool window = kb < end && (kb & 3) == 0;
      if (lane < P::SL)
        lds_dma<16>(sr, lds0 + (window ? P::XS + ((kb >> 2) & 1) * P::WINDOW + s0 * 16 : P::NONE),
                    window ? vs : kDmaOOB, (uint32_t)kb * 4);
    }
  };

  // ---- scales: a token's times the weight rows' ----
  const int nw = SW ? n0 + wn * 8 * NI : n0 + wn * 16 * NI;  // this wave's first row
  const bool idle = nw >= g.N;
  typedef const __attribute__((address_space(4))) float *scalar_t;  // scalar loads
  const scalar_t ws = (scalar_t)(g.ws + (size_t)rows.expert * g.ws_stride +
                                 (size_t)((idle ? n0 : nw) >> 7) * KB);
  constexpr int NS = SW ? 2 : 1;
  const uint32_t fs = lds0 + P::XS + (wm * NJ * 16 + l15) * 16;
  auto take_scales = [&](int kb, float (&to)[NS][NJ]) {
    const uint32_t at = fs + ((kb >> 2) & 1) * P::WINDOW + (kb & 3) * 4;
#pragma unroll
    for (int m = 0; m < NS; ++m) {
      const float f = ws[(size_t)m * NB * KB + kb];
#pragma unroll
      for (int j = 0; j < NJ; ++j) to[m][j] = lds_at<float>(at, j * 256) * f;
    }
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

  float s[NS][NJ];
#pragma unroll
  for (int t = 0; t + 1 < S; ++t)
#pragma unroll
    for (int q = 0; q < P::LOADS; ++q)
      load1(q, first + t, lds0 + t * P::STAGE, cut(first + t, 0), cut(first + t, 1));
  dma_wait_barrier<(S - 2) * P::LOADS>();
  take_scales(first, s);
#pragma unroll
  for (int j = 0; j < NJ; ++j) read_b(0, j);
  read_a(0, 0, 0);
  constexpr int LAG = 3;  // MFMAs between one and the use of its result
  f32x4_t p[LAG + 1];
  uint32_t base = 0, last = (S - 1) * P::STAGE;  // stages of this block, of the one before
  // a wave without tokens only loads and waits with the others
  if (wm * NJ * 16 >= rows.count) {
    for (int kb = first; kb < end; ++kb) {
      const bool even = cut(kb + S - 1, 0), odd = cut(kb + S - 1, 1);
#pragma unroll
      for (int q = 0; q < P::LOADS; ++q) load1(q, kb + S - 1, lds0 + last, even, odd);
      dma_wait_barrier<(S - 2) * P::LOADS>();
      last = base;
      base = base + P::STAGE == S * P::STAGE ? 0 : base + P::STAGE;
    }
  } else
  for (int kb = first; kb < end; ++kb) {
    const uint32_t next = base + P::STAGE == S * P::STAGE ? 0 : base + P::STAGE;
    const bool even = cut(kb + S - 1, 0), odd = cut(kb + S - 1, 1);
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
        dma_wait_barrier<(S - 2) * P::LOADS>();
        take_scales(kb + 1 < end ? kb + 1 : kb, sn);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int slot = i * NJ + j;
        if constexpr (EXACT)
          p[slot % (LAG + 1)] = mfma_codes(a[i & 1], b[j], f32x4_t{0.f, 0.f, 0.f, 0.f});
        else
          p[slot % (LAG + 1)] = mfma_fp8(a[i & 1], b[j]);
        __builtin_amdgcn_sched_barrier(0);
        if (slot >= LAG) add(slot - LAG);
        // the stage of the block before takes the loads of S - 1 blocks ahead, PER a pass
        constexpr int PER = NI - 1 >= P::LOADS ? 1 : 2 * (NI - 1) >= P::LOADS ? 2 : 4;
        static_assert(PER * (NI - 1) >= P::LOADS && NJ % PER == 0, "loads");
        if (j % (NJ / PER) == 0 && i + 1 < NI && i * PER + j / (NJ / PER) < P::LOADS)
          load1(i * PER + j / (NJ / PER), kb + S - 1, lds0 + last, even, odd);
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
    last = base;
    base = next;
  }

  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing may land in LDS after the end
  if constexpr (SW) {
    // h in place of the gates; a token's 128 columns are one group of the codes
    constexpr int NH = NI / 2;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < NH; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          acc[i][j][v] = silu_f32(acc[i][j][v]) * acc[i + NH][j][v];
          top = fmaxf(top, fabsf(acc[i][j][v]));
        }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (c == 0) tops[wn][(wm * NJ + j) * 16 + l15] = top;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int r = (wm * NJ + j) * 16 + l15;
      if (r >= rows.count) continue;
      const size_t row = (size_t)rows.row0 + r;
      float top = tops[0][r];
#pragma unroll
      for (int q = 1; q < WN; ++q) top = fmaxf(top, tops[q][r]);
      const Fp8Div d = fp8_div(top);
      if (wn == 0 && c == 0) g.ys[row * g.ld_ys + (n0 >> 7)] = d.scale;
      uint8_t *y = static_cast<uint8_t *>(g.y) + row * g.N + nw + 4 * c;
#pragma unroll
      for (int i = 0; i < NH; ++i)
        if (nw + 16 * i + 4 * c < g.N) {  // (N is a multiple of 16)
          const f32x4_t h = acc[i][j];
          *reinterpret_cast<uint32_t *>(y + 16 * i) =
              fp8_pack4(fp8_quotient(d, h[0]), fp8_quotient(d, h[1]), fp8_quotient(d, h[2]),
                        fp8_quotient(d, h[3]));
        }
    }
  } else {
    if (idle) return;
    if (g.kper) {  // partial sums [slices, M, N], f32
      g.y = g.part + (size_t)blockIdx.y * g.M * g.N;
      g.out_f32 = 1;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int r = (wm * NJ + j) * 16 + l15;
      if (r >= rows.count) continue;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        store4(g, (size_t)rows.row0 + r, nw + 16 * i + 4 * c, acc[i][j]);
    }
  }
}

// Sums the slices' partials in order: four neighbouring outputs per thread.
template <bool F32>
__global__ __launch_bounds__(256) void fp8_slices_kernel(const float *part, size_t n, int slices,
                                                         void *y) {
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int left = n - i < 4 ? (int)(n - i) : 4;
  float v[4] = {};
  if (left == 4 && n % 4 == 0) {
    f32x4_t t = *reinterpret_cast<const f32x4_t *>(part + i);
    for (int s = 1; s < slices; ++s) t += *reinterpret_cast<const f32x4_t *>(part + s * n + i);
    for (int q = 0; q < 4; ++q) v[q] = t[q];
  } else {
    for (int s = 0; s < slices; ++s)
      for (int q = 0; q < left; ++q) v[q] += part[s * n + i + q];
  }
  if (F32) {
    float *to = static_cast<float *>(y) + i;
    if (left == 4 && ((uintptr_t)to & 15) == 0)
      *reinterpret_cast<f32x4_t *>(to) = f32x4_t{v[0], v[1], v[2], v[3]};
    else
      for (int q = 0; q < left; ++q) to[q] = v[q];
  } else {
    uint16_t *to = static_cast<uint16_t *>(y) + i;
    const u32x2_t b = {f32_to_bf16_rne(v[0]) | (f32_to_bf16_rne(v[1]) << 16),
                       f32_to_bf16_rne(v[2]) | (f32_to_bf16_rne(v[3]) << 16)};
    if (left == 4 && ((uintptr_t)to & 7) == 0)
      *reinterpret_cast<u32x2_t *>(to) = b;
    else
      for (int q = 0; q < left; ++q) to[q] = (uint16_t)(b[q >> 1] >> (16 * (q & 1)));
  }
}

// Weight rows [n_first, n_first + count); count -1: all.
template <int NI, int NJ, int WN, int WM, bool SW, bool EXACT, int S>
hipError_t launch(const Fp8Gemm &g, hipStream_t st, int n_first = 0, int count = -1) {
  using P = Tile<NI, NJ, WN, WM, SW, S>;
  const int nt = ((count < 0 ? g.N : count) + P::OUT - 1) / P::OUT;
  const int slices = g.kper ? (fp8_blocks(g.K) + g.kper - 1) / g.kper : 1;
  const size_t tiles = (size_t)nt * (g.chunks ? g.max_chunks : (g.M + P::BM - 1) / P::BM);
  if (!launch_fits(tiles + 7, 64 * P::W)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fp8_tile_kernel<NI, NJ, WN, WM, SW, EXACT, S>),
                     dim3((unsigned)((tiles + 7) / 8 * 8), slices), dim3(64 * P::W), 0, st, g,
                     n_first, nt);
  if (slices > 1) {
    const size_t n = (size_t)g.M * g.N;
    const dim3 grid((unsigned)((n + 1023) / 1024));
    if (g.out_f32)
      hipLaunchKernelGGL(fp8_slices_kernel<true>, grid, dim3(256), 0, st, g.part, n, slices, g.y);
    else
      hipLaunchKernelGGL(fp8_slices_kernel<false>, grid, dim3(256), 0, st, g.part, n, slices, g.y);
  }
  return hipGetLastError();
}

constexpr int kCUs = 256;

// Slices of K for a product whose 128 x 128 tiles are fewer than the CUs take (two
// each): a multiple of 4 blocks per slice, 0 where one slice is left.  A workgroup's
// start and end weigh as much as some 8 blocks, so that is the least, unless 4 leave
// half the CUs idle; none where all of a short K fills half of them.  Measured, us, least 4 / 8, bf16 out: N x K 576 x 7168, 65 rows 15.0
// / 14.7 (f32 out 15.1 / 16.9), 512 21.8 / 19.2; 1536 x 7168, 333 27.0 / 22.9; 576 x
// 14336, 128 23.2 / 19.8; two slices / one: 7168 x 2048, 333 25.3 / 19.5, 512 26.3 / 20.6.
int slice_blocks(int M, int N, int K) {
  const int KB = fp8_blocks(K), tiles = fp8_blocks(M) * fp8_blocks(N);
  const int want = tiles >= 512 ? 1 : 512 / tiles;
  if (tiles > kCUs / 2 && KB <= 16) return 0;
  const int least = (int64_t)tiles * ((KB + 3) / 4) <= kCUs / 2 ? 4 : 8;
  const int even = ((KB + want - 1) / want + 3) & ~3, per = even > least ? even : least;
  return per < KB ? per : 0;
}

// The next larger tiles once the smaller ones take more than a round over the CUs.
// Measured, us, K = 4096, bf16 out, 128 x 128 / 256 x 128: 4096 x 1024 (256 / 128
// tiles) 38.3 / 36.7 (f32 out 52.8 / 63.0), 2048 x 2304 (288 / 144) 41.9 / 38.0 (f32
// out 71.7 / 65.7); 256 x 128 / 256 x 256: 4096 x 2048 (256 / 128) 41.5 / 58.0, 3328 x
// 3328 (338 / 169) 71.0 / 58.7.  (256 x 256 with f32 outputs: too few registers.)
Fp8Form tile_size(int M, int N, bool out_f32) {
  const int64_t middle = (int64_t)((N + 255) / 256) * fp8_blocks(M);
  return !out_f32 && middle > kCUs ? kFp8Tiles256
         : middle > kCUs / 2       ? kFp8Tiles256x128
                                   : kFp8Tiles128;
}

// Weight rows whose tiles of 256 x bm would fill at most half of a last round over
// the CUs: in tiles of half the size they fill twice as many, in a launch of their
// own.  Measured, us, one launch / two: bf16 out, 256 x 256, K = 4096, N x M: 4352 x
// 4096 (272 tiles) 114 / 97, 12000 x 1500 (282) 112 / 96, 14336 x 4096 (896) 263 / 243;
// f32 out, 256 x 128: 4352 x 4096 (544) 173 / 161, 4096 x 2100 (272) 116 / 104.
int last_round(int M, int N, int bm) {
  const int nt = (N + 255) / 256, mt = (M + bm - 1) / bm;
  const int full = (int)((int64_t)nt * mt / kCUs * kCUs / mt);  // n tiles of whole rounds
  if (full == 0 || full == nt || (int64_t)(nt - full) * mt > kCUs / 2) return 0;
  return N - full * 256;
}

}  // namespace

size_t fp8_partial_bytes(int M, int N, int K) {
  size_t most = 0;  // over all calls of up to M rows
  for (int m = 1; m <= fp8_blocks(M) && m * fp8_blocks(N) < 512; ++m) {
    const int rows = m * 128 < M ? m * 128 : M, per = slice_blocks(rows, N, K);
    if (!per || tile_size(rows, N, true) != kFp8Tiles128) continue;
    const size_t b = (size_t)((fp8_blocks(K) + per - 1) / per) * rows * N * 4;
    most = b > most ? b : most;
  }
  return most;
}

Fp8Form fp8_tile_form(int M, int N, int K, bool out_f32) {
  const Fp8Form f = tile_size(M, N, out_f32);
  return f == kFp8Tiles128 && slice_blocks(M, N, K) ? kFp8Slices128 : f;
}

// Fitted to the products named at fp8_form (off 7 to 18 % by form).  In slices: 0.75
// us per block of K of one, and the writing and joining of the partial sums, 2.5 us a
// million.
float fp8_tile_us(int M, int N, int K, bool out_f32) {
  const float KB = (float)fp8_blocks(K);
  switch (fp8_tile_form(M, N, K, out_f32)) {
    case kFp8Slices128: {
      const int per = slice_blocks(M, N, K), slices = (fp8_blocks(K) + per - 1) / per;
      return 10.0f + 0.75f * per + 2.5e-6f * M * N * slices;
    }
    case kFp8Tiles128:
      return 8.0f + KB * (0.6f + 0.5f * fp8_blocks(M) * fp8_blocks(N) / kCUs);
    case kFp8Tiles256x128:
      // (one round's; with more of them 32 x 32 takes far longer)
      return 12.0f + KB * (out_f32 ? 1.7f : 0.95f);
    default: {
      const int64_t tiles = (int64_t)((M + 255) / 256) * ((N + 255) / 256);
      return 18.0f + 0.7f * KB * (float)((tiles + kCUs - 1) / kCUs);
    }
  }
}

hipError_t fp8_tile_gemm(const Fp8Gemm &g0, hipStream_t st) {
  Fp8Gemm g = g0;
  g.kper = 0;
  if (g.swiglu)
    return g.exact ? launch<4, 4, 4, 2, true, true, 3>(g, st)
                   : launch<8, 2, 2, 4, true, false, 3>(g, st);
  if (g.chunks)
    return g.exact ? launch<4, 4, 4, 2, false, true, 3>(g, st)
                   : launch<8, 2, 2, 4, false, false, 3>(g, st);
  const Fp8Form f = fp8_tile_form(g.M, g.N, g.K, g.out_f32);
  if (f == kFp8Tiles256) {
    const int left = last_round(g.M, g.N, 256), most = g.N - left;
    const hipError_t e = launch<8, 4, 2, 4, false, false, 2>(g, st, 0, most);
    return e != hipSuccess || !left ? e : launch<8, 2, 2, 4, false, false, 3>(g, st, most, left);
  }
  if (f == kFp8Tiles256x128) {
    if (!g.out_f32) return launch<8, 2, 2, 4, false, false, 3>(g, st);
    // (exact: waves of 64 x 64 convert a fifth fewer codes than of 128 x 32)
    const int left = last_round(g.M, g.N, 128), most = g.N - left;
    const hipError_t e = launch<4, 4, 4, 2, false, true, 3>(g, st, 0, most);
    return e != hipSuccess || !left ? e : launch<4, 2, 2, 4, false, true, 2>(g, st, most, left);
  }
  if (f == kFp8Slices128) g.kper = slice_blocks(g.M, g.N, g.K);
  if (g.out_f32) return launch<4, 2, 2, 4, false, true, 2>(g, st);
  return launch<4, 2, 2, 4, false, false, 2>(g, st);
}

}  // namespace cai4
