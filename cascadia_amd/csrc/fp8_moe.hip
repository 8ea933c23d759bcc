// fp8_moe.hip -- one layer's experts in e4m3.
//
// Per token t and slot j with weight w >= threshold and an expert id inside the
// layer: h = silu(W_gate x) (W_up x) in f32 over x's codes, requantised, and
// y = bf16(W_down h); out_t = residual_t + sum_j w_j y_j in slot order (multiply,
// then add), rounded once.  y is kept in 16 bits between its product and the
// sum, as the INT4 layer keeps it: the slots' rows are the layer's largest
// intermediate (top_k times its output), and their rounding is no coarser than
// that of a bf16 output.
//
// Rows are grouped by expert (moe_group): position in a group varies between
// calls, results do not, since a grouped row's products do not depend on its
// place and the sum reads slots in order.
#include "fp8.hpp"
#include "fp8_common.hpp"
#include "moe.hpp"

namespace cai4 {
namespace {

// Rows of a chunk: the tile kernel's from a mean of 16 rows per expert.
int chunk_rows(int T, int E, int top_k) {
  return (int64_t)T * top_k >= (int64_t)16 * E ? kFp8TileRows : 16;
}

struct Layout {
  size_t xq, xs, pos, row_map, chunks, counts, h, hq, hs, y, total;
  int max_chunks, chunk_rows;
};

Layout layout_of(int H, int I, int E, int top_k, int T) {
  Layout w{};
  const size_t n = (size_t)T * top_k;
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 255) & ~(size_t)255;
    return at;
  };
  w.chunk_rows = chunk_rows(T, E, top_k);
  w.max_chunks = moe_max_chunks(T, E, top_k, w.chunk_rows);
  w.xq = take((size_t)T * H);
  w.xs = take((size_t)T * fp8_blocks(H) * 4);
  w.pos = take(n * 4);
  w.row_map = take(n * 4);
  w.chunks = take((size_t)w.max_chunks * sizeof(SkinnyChunk));
  w.counts = take(16);
  w.h = take(n * I * 4);
  w.hq = take(n * I);
  w.hs = take(n * fp8_blocks(I) * 4);
  w.y = take(n * H * 2);
  w.total = o;
  return w;
}

CAI4_DEV f32x4_t load4(const void *p, size_t at, bool f32) {
  if (f32) return *reinterpret_cast<const f32x4_t *>(static_cast<const float *>(p) + at);
  const u32x2_t v = *reinterpret_cast<const u32x2_t *>(static_cast<const uint16_t *>(p) + at);
  return f32x4_t{bitsf(v.x << 16), bitsf(v.x & 0xFFFF0000u), bitsf(v.y << 16),
                 bitsf(v.y & 0xFFFF0000u)};
}

// Four outputs of a token per thread (H is a multiple of 16).
__global__ __launch_bounds__(256) void fp8_combine_kernel(const void *residual, const uint16_t *y,
                                                          const int32_t *pos, const float *w,
                                                          int H, int k, void *out, int out_f32) {
#pragma clang fp contract(off)
  const int t = blockIdx.x, j = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (j >= H) return;
  const size_t o = (size_t)t * H + j;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < k; ++s) {
    const int p = pos[(size_t)t * k + s];
    if (p < 0) continue;
    v += w[(size_t)t * k + s] * load4(y, (size_t)p * H + j, false);
  }
  if (residual) v = load4(residual, o, out_f32) + v;
  if (out_f32) {
    *reinterpret_cast<f32x4_t *>(static_cast<float *>(out) + o) = v;
  } else {
    u32x2_t b;
    b.x = f32_to_bf16_rne(v.x) | (f32_to_bf16_rne(v.y) << 16);
    b.y = f32_to_bf16_rne(v.z) | (f32_to_bf16_rne(v.w) << 16);
    *reinterpret_cast<u32x2_t *>(static_cast<uint16_t *>(out) + o) = b;
  }
}

}  // namespace

size_t fp8_moe_workspace(int H, int I, int E, int top_k, int T) {
  return layout_of(H, I, E, top_k, T).total;
}

hipError_t fp8_moe_forward(const Fp8Moe &m, void *workspace, hipStream_t st) {
  const Layout w = layout_of(m.H, m.I, m.E, m.top_k, m.T);
  uint8_t *b = static_cast<uint8_t *>(workspace);
  uint8_t *xq = b + w.xq, *hq = b + w.hq;
  float *xs = reinterpret_cast<float *>(b + w.xs), *hs = reinterpret_cast<float *>(b + w.hs);
  int32_t *pos = reinterpret_cast<int32_t *>(b + w.pos);
  int32_t *row_map = reinterpret_cast<int32_t *>(b + w.row_map);
  SkinnyChunk *chunks = reinterpret_cast<SkinnyChunk *>(b + w.chunks);
  const int n = m.T * m.top_k, hb = fp8_blocks(m.H), ib = fp8_blocks(m.I);
  hipError_t e = fp8_quantize_rows(m.x, m.x_f32, m.T, m.H, xq, xs, st);
  if (e != hipSuccess) return e;
  e = moe_group(m.ids, m.weights, m.threshold, m.T, m.E, m.top_k, w.chunk_rows, w.max_chunks, pos,
                row_map, chunks, reinterpret_cast<int32_t *>(b + w.counts), st);
  if (e != hipSuccess) return e;
  Fp8Gemm g{};
  g.w = m.gate_up;
  g.ws = m.gate_up_s;
  g.x = xq;
  g.xs = xs;
  g.y = b + w.h;
  g.N = m.I;
  g.K = m.H;
  g.M = n;
  g.out_f32 = 1;
  g.chunks = chunks;
  g.max_chunks = w.max_chunks;
  g.chunk_rows = w.chunk_rows;
  g.n_chunks = reinterpret_cast<const int32_t *>(b + w.counts) + 1;
  g.x_rows = m.T;
  g.row_map = row_map;
  g.w_stride = (size_t)2 * m.I * m.H;
  g.ws_stride = (size_t)2 * ib * hb;
  g.swiglu = 1;
  e = fp8_gemm(g, st);
  if (e != hipSuccess) return e;
  e = fp8_quantize_rows(b + w.h, true, n, m.I, hq, hs, st);
  if (e != hipSuccess) return e;
  g.w = m.down;
  g.ws = m.down_s;
  g.x = hq;
  g.xs = hs;
  g.y = b + w.y;
  g.N = m.H;
  g.K = m.I;
  g.out_f32 = 0;
  g.row_map = nullptr;
  g.w_stride = (size_t)m.H * m.I;
  g.ws_stride = (size_t)hb * ib;
  g.swiglu = 0;
  e = fp8_gemm(g, st);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fp8_combine_kernel, dim3(m.T, (m.H + 1023) / 1024), dim3(256), 0, st,
                     m.residual, reinterpret_cast<const uint16_t *>(b + w.y), pos, m.weights, m.H,
                     m.top_k, m.out, m.out_f32);
  return hipGetLastError();
}

}  // namespace cai4
