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
// (exact) give 1e-8.  The kernels here stream weights (of some hundred rows they wait
// for them), so that the products run on the bf16 MFMAs, codes converted in registers.
//
// Bound: HBM, every weight read once per 16 or 32 rows of x (of more rows: the
// conversion of codes, and latency).  A workgroup's
// waves take the k-blocks of its rows in turn, so that together they read
// contiguous kilobytes of each row; their sums are added through LDS in wave order.
// Measured: 14336 x 4096, 16 rows 16 us (3.7 TB/s); 60 experts of 3584 x 1408 with 256
// rows in all: gate and up 94 us (5.3 TB/s of the codes that rows meet); one row of 4096
// x 4096 6.6 us (on another card 9.3), one token's 8 experts of 7168 x 2048 46.6 us (5.0
// TB/s) and 30.0 us.  A row whose codes are in hand takes fp8_few_kernel: 8.4 us a call
// with weights from HBM, a bf16 row 9.1.
#include "fp8.hpp"
#include "fp8_common.hpp"
#include "fp8_rows.hpp"
#include "lds_dma.hpp"
#include "moe_route.hpp"

namespace cai4 {
namespace {

// 16 bytes at byte `off` (zeros past the range).
CAI4_DEV u32x4_t load16(rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

typedef const __attribute__((address_space(4))) float *scalar_t;  // scalar loads

// 16 weight rows from n0 on of matrix m (SwiGLU: 0 gate, 1 up), as a wave streams them.
struct Weights {
  rsrc_t r;
  scalar_t ws;
  int rows;
  uint32_t row, block;  // bytes between rows, between blocks of K
};
CAI4_DEV Weights weights_of(const Fp8Gemm &g, int expert, int n0, int m) {
  const int KB = (g.K + 127) >> 7, NB = (g.N + 127) >> 7;
  Weights w;
  w.rows = n0 >= g.N ? 0 : g.N - n0 < 16 ? g.N - n0 : 16;
  const int n = w.rows ? n0 : 0;
  const uint8_t *p = g.w + (size_t)expert * g.w_stride;
  if (g.w_tiled) {
    const size_t band = KB * kFp8BlockBytes, in = (size_t)(n & 127) * 128;
    w.r = rsrc_scalar(p + ((size_t)m * NB + (n >> 7)) * band + in, w.rows ? band - in : 0);
    w.row = 128;
    w.block = kFp8BlockBytes;
  } else {
    w.r = rsrc_scalar(p + ((size_t)m * g.N + n) * g.K, (size_t)w.rows * g.K);
    w.row = g.K;
    w.block = 128;
  }
  w.ws = (scalar_t)(g.ws + (size_t)expert * g.ws_stride + ((size_t)m * NB + (n >> 7)) * KB);
  return w;
}
// This lane's two chunks of block kb (past the rows or columns: zeros).
CAI4_DEV void load_weights(const Weights &w, int kb, int K, int l15, int c, u32x4_t (&a)[2]) {
  const uint32_t at = (uint32_t)l15 * w.row + (uint32_t)kb * w.block + 16 * c;
  const int c0 = kb * 128 + 16 * c;
  a[0] = load16(w.r, l15 < w.rows && c0 < K ? at : kDmaOOB);
  a[1] = load16(w.r, l15 < w.rows && c0 + 64 < K ? at + 64 : kDmaOOB);
}

// 16 MT weight rows (SW: the same 16 of gate and of up) x 16 NT rows of x per
// workgroup.  The scales of x, whose rows lie apart, go to LDS once per window of
// blocks: read per block they were a third of all requests.
constexpr int kFewWindow = 128;

template <int NT, bool SW>
__global__ __launch_bounds__(512) void fp8_few_kernel(Fp8Gemm g) {
  constexpr int W = 8, MT = 2, OUT = SW ? 16 : 32;
  __shared__ f32x4_t part[W][MT * NT][64];
  __shared__ float scales[kFewWindow][16 * NT];
  const int lane = threadIdx.x & 63, l15 = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ntiles = (g.N + OUT - 1) / OUT, mt = blockIdx.x / ntiles;
  if (g.chunks && mt >= *g.n_chunks) return;  // the whole workgroup
  const Rows rows = rows_of(g, mt, 16 * NT);
  const int n0 = (blockIdx.x - mt * ntiles) * OUT;
  const int KB = (g.K + 127) >> 7;
  Weights w[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    w[m] = weights_of(g, rows.expert, SW ? n0 : n0 + 16 * m, SW ? m : 0);
  const rsrc_t xr = g.row_map ? rsrc_scalar(g.x, (size_t)g.x_rows * g.K)
                              : rsrc_scalar(g.x + (size_t)rows.row0 * g.K,
                                            (size_t)rows.count * g.K);
  uint32_t xo[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = 16 * t + l15;
    xo[t] = r >= rows.count ? kDmaOOB
            : (g.row_map ? (uint32_t)g.row_map[rows.row0 + r] : (uint32_t)r) * (uint32_t)g.K;
  }
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < KB; k0 += kFewWindow) {
    const int k1 = KB - k0 < kFewWindow ? KB : k0 + kFewWindow;
    if (k0) __syncthreads();
    // 32 lanes along a row, 16 rows at a time
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = 16 * t + (int)(threadIdx.x >> 5), row = rows.row0 + r;
      const bool in = r < rows.count;
      const float *s = g.xs + (size_t)(in ? g.row_map ? g.row_map[row] : row : 0) * g.ld_xs;
      for (int k = k0 + (int)(threadIdx.x & 31); k < k1; k += 32)
        scales[k - k0][r] = in ? s[k] : 0.f;
    }
    __syncthreads();
    // (many waves with one block each in flight: loads ahead of the block, or two
    // batches of them, cost registers and measured slower)
    for (int kb = k0 + wave; kb < k1; kb += W) {
      const int c0 = kb * 128 + 16 * c, c1 = c0 + 64;
      u32x4_t a[MT][2], b[NT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) load_weights(w[m], kb, g.K, l15, c, a[m]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        b[t][0] = load16(xr, xo[t] != kDmaOOB && c0 < g.K ? xo[t] + c0 : kDmaOOB);
        b[t][1] = load16(xr, xo[t] != kDmaOOB && c1 < g.K ? xo[t] + c1 : kDmaOOB);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float f = w[m].ws[kb];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const f32x4_t p = mfma_codes(a[m], b[t], f32x4_t{0.f, 0.f, 0.f, 0.f});
          const float s = scales[kb - k0][16 * t + l15] * f;
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][t][i] = __fmaf_rn(p[i], s, acc[m][t][i]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][m * NT + t][lane] = acc[m][t];
  __syncthreads();
  if (wave >= (SW ? NT : MT * NT)) return;
  const int t = wave % NT;
  f32x4_t v = part[0][wave][lane];
#pragma unroll
  for (int q = 1; q < W; ++q) v += part[q][wave][lane];
  if (SW) {
    f32x4_t u = part[0][wave + NT][lane];
#pragma unroll
    for (int q = 1; q < W; ++q) u += part[q][wave + NT][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = silu_f32(v[i]) * u[i];
  }
  const int n = n0 + 16 * (wave / NT) + 4 * c;
  if (16 * t + l15 < rows.count && n < g.N)
    store4(g, (size_t)rows.row0 + 16 * t + l15, n, v);
}

// ---------------------------------------------------------------------------
// one row, quantised here
// ---------------------------------------------------------------------------

constexpr int kOneBlocks = 128;  // blocks of the row in LDS: K up to 16,384

// Blocks first, first + step, ... of a bf16 or f32 row as codes and scales in LDS,
// by one wave, two columns per lane; U blocks at a time, so that their loads and
// their reductions overlap.
template <bool F32, int U>
CAI4_DEV void quantize_row(const void *x, int K, int first, int step, int lane,
                           uint8_t (*codes)[128], float *scales) {
  const int KB = (K + 127) >> 7;
  // buffer loads, out of range past the end: a branch around each would wait for it
  const rsrc_t r = rsrc(x, (size_t)K * (F32 ? 4 : 2));
  for (int k0 = first; k0 < KB; k0 += U * step) {
    float v[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t col = (uint32_t)(k0 + u * step) * 128 + 2 * lane;
      if (F32) {
        const auto d = __builtin_amdgcn_raw_buffer_load_b64(r, col * 4, 0, 0);
        v[u][0] = bitsf((uint32_t)d[0]);
        v[u][1] = bitsf((uint32_t)d[1]);
      } else {
        const uint32_t d = __builtin_amdgcn_raw_buffer_load_b32(r, col * 2, 0, 0);
        v[u][0] = bitsf(d << 16);
        v[u][1] = bitsf(d & 0xFFFF0000u);
      }
    }
    float top[U];
#pragma unroll
    for (int u = 0; u < U; ++u) top[u] = wave_max_f32(fmaxf(fabsf(v[u][0]), fabsf(v[u][1])));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = k0 + u * step;
      if (kb >= KB) break;  // uniform
      const Fp8Div d = fp8_div(top[u]);
      const int q = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_quotient(d, v[u][0]),
                                                    fp8_quotient(d, v[u][1]), 0, false);
      *reinterpret_cast<uint16_t *>(&codes[kb][2 * lane]) = (uint16_t)q;
      if (lane == 0) scales[kb] = d.scale;
    }
  }
}

// MT sets of 16 weight rows times the row of x in LDS, this wave's blocks first,
// first + step, ..., two of them in flight (four: slower).  The tokens' operand
// holds the row in all 16 columns.
template <int MT, class Row>
CAI4_DEV void stream_row(const Weights (&w)[MT], int K, int first, int step, int lane,
                         const uint8_t (*codes)[128], const float *scales, f32x4_t (&acc)[MT],
                         Row row) {
  const int l15 = lane & 15, c = lane >> 4, KB = (K + 127) >> 7;
  u32x4_t a[2][MT][2];
  auto load = [&](u32x4_t (&to)[MT][2], int kb) {  // (past the end: out of range)
#pragma unroll
    for (int m = 0; m < MT; ++m) load_weights(w[m], kb, K, l15, c, to[m]);
  };
  auto add = [&](const u32x4_t (&from)[MT][2], int kb) {
    const u32x4_t b[2] = {*reinterpret_cast<const u32x4_t *>(&codes[kb][16 * c]),
                          *reinterpret_cast<const u32x4_t *>(&codes[kb][64 + 16 * c])};
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const f32x4_t p = mfma_codes(from[m], b, f32x4_t{0.f, 0.f, 0.f, 0.f});
      const float s = scales[kb] * w[m].ws[kb];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] = __fmaf_rn(p[i], s, acc[m][i]);
    }
  };
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  load(a[0], first);
  load(a[1], first + step);
  row();  // the row is quantised while the first weights are on their way
  int kb = first;
  for (; kb + step < KB; kb += 2 * step) {
    add(a[0], kb);
    load(a[0], kb + 2 * step);
    add(a[1], kb + step);
    load(a[1], kb + 3 * step);
  }
  if (kb < KB) add(a[0], kb);
}

CAI4_DEV bool slot_in(const int32_t *ids, const float *weights, float threshold, int E, int s) {
  return !(weights[s] < threshold) && ids[s] >= 0 && ids[s] < E;
}

// y = W x for one row of x; SW: h = silu(gate x) (up x), f32, for the experts of
// one token's slots (blockIdx.y: the slot).  16 outputs per workgroup.
template <bool SW, bool F32>
__global__ __launch_bounds__(512) void fp8_one_kernel(Fp8Gemm g, const void *x,
                                                      const int32_t *ids, const float *weights,
                                                      float threshold, int E) {
  constexpr int W = 8, MT = SW ? 2 : 1;
  __shared__ f32x4_t part[W][MT][4];
  __shared__ __attribute__((aligned(16))) uint8_t codes[kOneBlocks][128];
  __shared__ float scales[kOneBlocks];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, slot = blockIdx.y;
  if (SW && !slot_in(ids, weights, threshold, E, slot)) return;  // the whole workgroup
  const int e = SW ? __builtin_amdgcn_readfirstlane(ids[slot]) : 0;
  Weights w[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) w[m] = weights_of(g, e, n0, m);
  f32x4_t acc[MT];
  stream_row<MT>(w, g.K, wave, W, lane, codes, scales, acc, [&]() {
    quantize_row<F32, 4>(x, g.K, wave, W, lane, codes, scales);
    __syncthreads();
  });
  if ((lane & 15) == 0) {
#pragma unroll
    for (int m = 0; m < MT; ++m) part[wave][m][lane >> 4] = acc[m];
  }
  __syncthreads();
  if (threadIdx.x >= 4) return;
  f32x4_t v[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    v[m] = part[0][m][threadIdx.x];
#pragma unroll
    for (int q = 1; q < W; ++q) v[m] += part[q][m][threadIdx.x];
  }
  if (SW) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[0][i] = silu_f32(v[0][i]) * v[MT - 1][i];
  }
  if (n0 + 4 * (int)threadIdx.x < g.N) store4(g, slot, n0 + 4 * threadIdx.x, v[0]);
}

// The down products of one token's slots and their weighted sum: 16 outputs per
// workgroup, `per` waves for each slot, each slot's row in a part of the LDS.
__global__ __launch_bounds__(1024) void fp8_one_down_kernel(Fp8Gemm g, const float *h,
                                                            const int32_t *ids,
                                                            const float *weights, float threshold,
                                                            int E, int top_k, int per,
                                                            const void *residual) {
#pragma clang fp contract(off)
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ f32x4_t part[16][4];
  const int KB = (g.K + 127) >> 7;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, slot = wave / per, first = wave - slot * per;
  uint8_t(*codes)[128] = reinterpret_cast<uint8_t(*)[128]>(lds + (size_t)slot * KB * 128);
  float *scales = reinterpret_cast<float *>(lds + (size_t)top_k * KB * 128) + slot * KB;
  const bool in = slot_in(ids, weights, threshold, E, slot);
  Weights w[1] = {weights_of(g, in ? __builtin_amdgcn_readfirstlane(ids[slot]) : 0, n0, 0)};
  if (!in) w[0].rows = 0;  // nothing is read, what is added up is not used
  f32x4_t acc[1];
  stream_row<1>(w, g.K, first, per, lane, codes, scales, acc, [&]() {
    if (in) quantize_row<true, 4>(h + (size_t)slot * g.K, g.K, first, per, lane, codes, scales);
    __syncthreads();
  });
  if ((lane & 15) == 0) part[wave][lane >> 4] = acc[0];
  __syncthreads();
  const int n = n0 + (int)threadIdx.x;
  if (threadIdx.x >= 16 || n >= g.N) return;
  float v = 0.f;
  for (int s = 0; s < top_k; ++s) {
    if (!slot_in(ids, weights, threshold, E, s)) continue;
    float y = 0.f;
    for (int q = 0; q < per; ++q)
      y += reinterpret_cast<const float *>(part[s * per + q])[threadIdx.x];
    v += weights[s] * y;
  }
  if (g.out_f32) {
    if (residual) v = static_cast<const float *>(residual)[n] + v;
    static_cast<float *>(g.y)[n] = v;
  } else {
    if (residual) v = bf16_to_f32(static_cast<const uint16_t *>(residual)[n]) + v;
    static_cast<uint16_t *>(g.y)[n] = (uint16_t)f32_to_bf16_rne(v);
  }
}

template <int NT, bool SW>
hipError_t few(const Fp8Gemm &g, hipStream_t st) {
  const int out = SW ? 16 : 32;
  const size_t tiles = (size_t)((g.N + out - 1) / out) *
                       (g.chunks ? g.max_chunks : (g.M + 16 * NT - 1) / (16 * NT));
  if (!launch_fits(tiles, 512)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fp8_few_kernel<NT, SW>), dim3((unsigned)tiles), dim3(512), 0, st, g);
  return hipGetLastError();
}

}  // namespace

// Estimated time of a product in 32 x 32 outputs per workgroup, us: a round over the
// CUs costs 0.2 us per block of K (off 10 % as a whole over 1,260 products of 17 to
// 1,024 rows, 246 to 24,576 x 272 to 14,336).
static float few_us(int M, int N, int K) {
  const int64_t groups = (int64_t)((N + 31) / 32) * ((M + 31) / 32);
  return 3.0f + (float)((groups + 255) / 256) * (0.2f * fp8_blocks(K) + 0.6f);
}

// Tiles where fp8_tile_us says less.  Measured, us, 32 x 32 / tiles, bf16 out (f32
// out), N x K: 4096 x 1024, 256 rows 13.0 / 14.8, 448 20.8 / 11.0 (20.4 / 14.0); 2395 x
// 272, 640 12.6 / 12.5, 1024 19.2 / 12.9; 576 x 7168, 96 16.3 / 14.0 (16.2 / 15.2), 333
// 16.8 / 16.8 (16.7 / 19.2), 512 29.1 / 18.6; 246 x 4336, 333 9.3 / 20.7; 1137 x 9152,
// 200 17.2 / 23.2, 512 41.6 / 33.1; 4096 x 4096, 96 19.2 / 17.2; 14336 x 4096, 32 21.9 /
// 19.2.  Over those products the choice costs 0.8 % more than the faster form of each.
Fp8Form fp8_form(int M, int N, int K, bool out_f32) {
  if (M <= kFp8FewRows) return kFp8Rows16;
  return fp8_tile_us(M, N, K, out_f32) < few_us(M, N, K) ? fp8_tile_form(M, N, K, out_f32)
                                                         : kFp8Rows32;
}

hipError_t fp8_gemm(const Fp8Gemm &g, hipStream_t st) {
  if (g.chunks) {
    if (g.chunk_rows > 16) return fp8_tile_gemm(g, st);
    return g.swiglu ? few<1, true>(g, st) : few<1, false>(g, st);
  }
  const Fp8Form f = fp8_form(g.M, g.N, g.K, g.out_f32);
  if (f == kFp8Rows16) return few<1, false>(g, st);
  return f == kFp8Rows32 ? few<2, false>(g, st) : fp8_tile_gemm(g, st);
}

bool fp8_one_row(int K) { return K <= kOneBlocks * 128; }

// One token's rows fit LDS: x's, and every slot's h.
bool fp8_one_token(int H, int I, int top_k) {
  return fp8_one_row(H) && (size_t)top_k * fp8_blocks(I) * 132 <= 48 * 1024;
}

hipError_t fp8_gemv(const Fp8Gemm &g, const void *x, bool x_f32, hipStream_t st) {
  const dim3 grid((g.N + 15) / 16), block(512);
  if (x_f32)
    hipLaunchKernelGGL((fp8_one_kernel<false, true>), grid, block, 0, st, g, x, nullptr, nullptr,
                       0.f, 0);
  else
    hipLaunchKernelGGL((fp8_one_kernel<false, false>), grid, block, 0, st, g, x, nullptr, nullptr,
                       0.f, 0);
  return hipGetLastError();
}

hipError_t fp8_moe_one(const Fp8Moe &m, const Fp8Gemm &gate_up, const Fp8Gemm &down, float *h,
                       hipStream_t st) {
  const dim3 grid((gate_up.N + 15) / 16, m.top_k), block(512);
  if (m.x_f32)
    hipLaunchKernelGGL((fp8_one_kernel<true, true>), grid, block, 0, st, gate_up, m.x, m.ids,
                       m.weights, m.threshold, m.E);
  else
    hipLaunchKernelGGL((fp8_one_kernel<true, false>), grid, block, 0, st, gate_up, m.x, m.ids,
                       m.weights, m.threshold, m.E);
  const int per = m.top_k >= 8 ? 1 : 8 / m.top_k;
  hipLaunchKernelGGL(fp8_one_down_kernel, dim3((down.N + 15) / 16), dim3(64 * per * m.top_k),
                     (size_t)m.top_k * fp8_blocks(down.K) * 132, st, down, h, m.ids, m.weights,
                     m.threshold, m.E, m.top_k, per, m.residual);
  return hipGetLastError();
}

}  // namespace cai4
