// fp8_moe.hip -- one layer's experts in e4m3.
//
// Per token t and slot j with weight w >= threshold and an expert id inside the
// layer: h = silu(W_gate x) (W_up x) in f32 over x's codes, requantised, and
// y = W_down h in f32; out_t = residual_t + sum_j w_j y_j in slot order (multiply,
// then add), rounded once.
//
// Rows are grouped by expert.  Position in a group varies between calls, results
// do not: a grouped row's products do not depend on its place, and the sum reads
// slots in order.
//
// One token: two launches, each quantising the rows it reads (fp8_gemm.hip).
// More: x's codes and, in workgroups of the same launch, the experts' counts
// (for up to 1,024 slots the whole grouping); the grouping; gate / up; h's codes
// (on tiles in the gate / up launch itself); down; the weighted sum.  2,048 tokens over
// 128 experts, 8 each: 8 + 9 us before the products, 56 for the sum (302 MB at 5.4
// TB/s); 32 over 60: 5 + 5 for h's codes + 5.5.  Slots' rows kept in 16 bits would take
// 32 us less (738 for 770 in all) and put the output 0.7e-3 off.
#include "fp8.hpp"
#include "fp8_common.hpp"
#include "fp8_quant.hpp"

namespace cai4 {
namespace {

// Rows of a chunk: the tile kernel's from a mean of 8 rows per expert.  Measured, us,
// 16-row chunks / tiles at a mean of 4, 8, 12 and 16 rows, bf16 out: 60 experts of 3584 x
// 1408, even 177 / 191, 196 / 198, 217 / 202, 262 / 206; Zipf 158 / 176, 209 / 198, 238 /
// 203, 271 / 209; 128 of 2048 x 1024, Zipf 138 / 132, 189 / 171, 232 / 181, 270 / 186.
// f32 out, at 8 and 12: 196 / 219, 218 / 222; 209 / 219, 239 / 230; 189 / 196, 232 / 203.
constexpr int kTileMean = 8;

// Workgroups that count: 1,024 slots each, at most 64 (a placing workgroup adds
// up all counts before its own).
constexpr int kCountSlots = 1024, kMaxCounters = 64;
int counters(size_t n) {
  const size_t b = (n + kCountSlots - 1) / kCountSlots;
  return b < (size_t)kMaxCounters ? (int)b : kMaxCounters;
}

// Counts in rows of whole 16 bytes.
__host__ __device__ inline int fp8_ld_experts(int E) { return (E + 3) & ~3; }

struct Layout {
  size_t xq, xs, pos, row_map, chunks, counts, hist, h, hq, hs, y, total;
  int max_chunks, chunk_rows, counters;
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
  w.chunk_rows = fp8_moe_chunk_rows(T, E, top_k);
  // sum of ceil(c_e / C) <= A + (n - A) / C for A experts with rows
  const size_t a = n < (size_t)E ? n : E;
  w.max_chunks = (int)(a + (n - a) / w.chunk_rows);
  w.counters = counters(n);
  w.xq = take((size_t)T * H);
  w.xs = take((size_t)T * fp8_ld(H) * 4);
  w.pos = take(n * 4);
  w.row_map = take(n * 4);
  w.chunks = take((size_t)w.max_chunks * sizeof(Fp8Chunk));
  w.counts = take(16);
  w.hist = take((size_t)w.counters * fp8_ld_experts(E) * 4);
  w.h = take(T > 1 && w.chunk_rows == kFp8TileRows ? 0 : n * I * 4);
  w.hq = take(n * I);
  w.hs = take(n * fp8_ld(I) * 4);
  w.y = take(n * H * 4);
  w.total = o;
  return w;
}

struct Group {
  const int32_t *ids;
  const float *weights;
  float threshold;
  int n, top_k, E, chunk_rows, counters;
  int32_t *pos, *row_map, *hist;  // hist: [counters, fp8_ld_experts(E)]
  Fp8Chunk *chunks;
  int32_t *n_chunks;
};

constexpr int kGroupThreads = 256, kPer = kRouteMaxExperts / kGroupThreads;
struct GroupLds {
  int cnt[kRouteMaxExperts];  // counts; then first rows
  int waves[2][4];
};

// The slots of counter b: [first, last).
CAI4_DEV void slots_of(const Group &g, int b, int &first, int &last) {
  const int per = (g.n + g.counters - 1) / g.counters;
  first = b * per;
  last = first + per < g.n ? first + per : g.n;
}

// Counts a share of the slots; pos[i] becomes slot i's rank among its expert's in
// the share, or -1 for a slot that is left out.
CAI4_DEV void count_slots(const Group &g, int b, GroupLds &l) {
  for (int e = threadIdx.x; e < g.E; e += kGroupThreads) l.cnt[e] = 0;
  __syncthreads();
  int first, last;
  slots_of(g, b, first, last);
  for (int i = first + (int)threadIdx.x; i < last; i += kGroupThreads) {
    const int e = g.ids[i];
    const bool in = !(g.weights[i] < g.threshold) && e >= 0 && e < g.E;
    g.pos[i] = in ? atomicAdd(&l.cnt[e], 1) : -1;
  }
  __syncthreads();
}

// Inclusive sum over the workgroup's threads of v.
CAI4_DEV int group_scan(int v, int *waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  for (int q = 0; q < wave; ++q) v += waves[q];
  return v;
}

// From the experts' counts over all slots (total) and over the shares before this
// one (before), kPer neighbouring experts per thread: first rows, chunks (by
// share 0), and the places of the share's slots.
CAI4_DEV void place_slots(const Group &g, int b, const int *total, const int *before,
                          GroupLds &l) {
  const int e0 = threadIdx.x * kPer;
  int rows = 0, chunks = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    rows += total[q];
    chunks += (total[q] + g.chunk_rows - 1) / g.chunk_rows;
  }
  int row = group_scan(rows, l.waves[0]) - rows;
  int chunk = group_scan(chunks, l.waves[1]) - chunks;
  __syncthreads();  // (counts read by every thread before they are replaced)
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int e = e0 + q, nc = (total[q] + g.chunk_rows - 1) / g.chunk_rows;
    if (e < g.E) {
      l.cnt[e] = row + before[q];
      if (b == 0)
        for (int i = 0; i < nc; ++i) {
          const int left = total[q] - i * g.chunk_rows;
          g.chunks[chunk + i] = Fp8Chunk{e, row + i * g.chunk_rows,
                                         left < g.chunk_rows ? left : g.chunk_rows, chunk, nc};
        }
    }
    row += total[q];
    chunk += nc;
  }
  if (b == 0 && threadIdx.x == kGroupThreads - 1) *g.n_chunks = chunk;
  __syncthreads();
  int first, last;
  slots_of(g, b, first, last);
  for (int i = first + (int)threadIdx.x; i < last; i += kGroupThreads) {
    const int rank = g.pos[i];
    if (rank < 0) continue;
    const int p = l.cnt[g.ids[i]] + rank;
    g.pos[i] = p;
    g.row_map[p] = i / g.top_k;
  }
}

// The first `counters` workgroups count (one alone: also places), the others
// quantise x.
template <bool F32>
__global__ __launch_bounds__(256) void fp8_moe_prep_kernel(Group g, const void *x, size_t groups,
                                                           int K, int KB, uint8_t *codes,
                                                           float *scales, int ld) {
  __shared__ GroupLds l;
  const int b = blockIdx.x;
  if (b >= g.counters) {
    quantize_rows_step<F32>((size_t)(b - g.counters), x, groups, K, KB, codes, scales, ld);
    return;
  }
  count_slots(g, b, l);
  const int e0 = threadIdx.x * kPer;
  if (g.counters == 1) {
    int total[kPer], before[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      total[q] = e0 + q < g.E ? l.cnt[e0 + q] : 0;
      before[q] = 0;
    }
    place_slots(g, 0, total, before, l);
  } else {
    // (kPer is 4: a thread's experts are one load)
    const int ld = fp8_ld_experts(g.E);
    for (int e = threadIdx.x; e < ld; e += kGroupThreads)
      g.hist[(size_t)b * ld + e] = e < g.E ? l.cnt[e] : 0;
  }
}

__global__ __launch_bounds__(256) void fp8_moe_place_kernel(Group g) {
  __shared__ GroupLds l;
  const int b = blockIdx.x, e0 = threadIdx.x * kPer;
  int total[kPer] = {}, before[kPer] = {};
  static_assert(kPer == 4, "one load per share");
  const int ld = fp8_ld_experts(g.E);
  if (e0 < g.E)
    for (int s0 = 0; s0 < g.counters; s0 += 8) {  // eight loads in flight
      u32x4_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int s = s0 + i < g.counters ? s0 + i : s0;
        v[i] = *reinterpret_cast<const u32x4_t *>(g.hist + (size_t)s * ld + e0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int c = s0 + i < g.counters ? (int)v[i][q] : 0;
          total[q] += c;
          before[q] += s0 + i < b ? c : 0;
        }
    }
  place_slots(g, b, total, before, l);
}

CAI4_DEV f32x4_t load4(const void *p, size_t at, bool f32) {
  if (f32) return *reinterpret_cast<const f32x4_t *>(static_cast<const float *>(p) + at);
  const u32x2_t v = *reinterpret_cast<const u32x2_t *>(static_cast<const uint16_t *>(p) + at);
  return f32x4_t{bitsf(v.x << 16), bitsf(v.x & 0xFFFF0000u), bitsf(v.y << 16),
                 bitsf(v.y & 0xFFFF0000u)};
}

// Four outputs of a token per thread (H is a multiple of 16).
__global__ __launch_bounds__(256) void fp8_combine_kernel(const void *residual, const float *y,
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
    v += w[(size_t)t * k + s] * load4(y, (size_t)p * H + j, true);
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

int fp8_moe_chunk_rows(int T, int E, int top_k) {
  return (int64_t)T * top_k >= (int64_t)kTileMean * E ? kFp8TileRows : 16;
}

bool fp8_moe_fits(int H, int I, int E, int top_k, int T) {
  const Layout w = layout_of(H, I, E, top_k, T);
  const bool tiles = w.chunk_rows == kFp8TileRows;
  const size_t up = tiles ? (I + 127) / 128 : (I + 15) / 16;
  const size_t down = tiles ? (H + 255) / 256 : (H + 31) / 32;
  return launch_fits((up > down ? up : down) * w.max_chunks + 7, 512);
}

size_t fp8_moe_workspace(int H, int I, int E, int top_k, int T) {
  size_t most = 0;  // over all calls of up to T tokens
  auto take = [&](int t) {
    const size_t bytes = layout_of(H, I, E, top_k, t).total;
    most = bytes > most ? bytes : most;
  };
  take(T);
  // (one token, and the largest batch in 16-row chunks, may need more than one on tiles)
  take(1);
  const int few = (int)(((int64_t)kTileMean * E - 1) / top_k);
  if (few >= 1 && few < T) take(few);
  return most;
}

hipError_t fp8_moe_forward(const Fp8Moe &m, void *workspace, hipStream_t st) {
  const Layout w = layout_of(m.H, m.I, m.E, m.top_k, m.T);
  uint8_t *b = static_cast<uint8_t *>(workspace);
  uint8_t *xq = b + w.xq, *hq = b + w.hq;
  float *xs = reinterpret_cast<float *>(b + w.xs), *hs = reinterpret_cast<float *>(b + w.hs);
  const int n = m.T * m.top_k, hb = fp8_blocks(m.H), ib = fp8_blocks(m.I);
  Fp8Gemm up{}, down{};
  up.w = m.gate_up;
  up.ws = m.gate_up_s;
  up.N = m.I;
  up.K = m.H;
  up.M = n;
  up.w_tiled = down.w_tiled = m.tiled;
  up.w_stride = 2 * (m.tiled ? fp8_tiled_bytes(m.I, m.H) : (size_t)m.I * m.H);
  up.ws_stride = (size_t)2 * ib * hb;
  up.swiglu = 1;
  up.out_f32 = 1;
  up.exact = down.exact = m.out_f32;
  down.w = m.down;
  down.ws = m.down_s;
  down.N = m.H;
  down.K = m.I;
  down.M = n;
  down.w_stride = m.tiled ? fp8_tiled_bytes(m.H, m.I) : (size_t)m.H * m.I;
  down.ws_stride = (size_t)hb * ib;

  if (m.T == 1 && fp8_one_token(m.H, m.I, m.top_k)) {
    float *h = reinterpret_cast<float *>(b + w.h);
    up.y = h;
    down.y = m.out;
    down.out_f32 = m.out_f32;
    return fp8_moe_one(m, up, down, h, st);
  }

  Group gr{};
  gr.ids = m.ids;
  gr.weights = m.weights;
  gr.threshold = m.threshold;
  gr.n = n;
  gr.top_k = m.top_k;
  gr.E = m.E;
  gr.chunk_rows = w.chunk_rows;
  gr.counters = w.counters;
  gr.pos = reinterpret_cast<int32_t *>(b + w.pos);
  gr.row_map = reinterpret_cast<int32_t *>(b + w.row_map);
  gr.hist = reinterpret_cast<int32_t *>(b + w.hist);
  gr.chunks = reinterpret_cast<Fp8Chunk *>(b + w.chunks);
  gr.n_chunks = reinterpret_cast<int32_t *>(b + w.counts);
  const size_t groups = (size_t)m.T * hb;
  const dim3 grid((unsigned)(w.counters + (groups + kRowGroups - 1) / kRowGroups));
  if (m.x_f32)
    hipLaunchKernelGGL(fp8_moe_prep_kernel<true>, grid, dim3(256), 0, st, gr, m.x, groups, m.H, hb,
                       xq, xs, fp8_ld(m.H));
  else
    hipLaunchKernelGGL(fp8_moe_prep_kernel<false>, grid, dim3(256), 0, st, gr, m.x, groups, m.H,
                       hb, xq, xs, fp8_ld(m.H));
  if (w.counters > 1)
    hipLaunchKernelGGL(fp8_moe_place_kernel, dim3(w.counters), dim3(256), 0, st, gr);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;

  const bool tiles = w.chunk_rows == kFp8TileRows;
  up.x = xq;
  up.xs = xs;
  up.ld_xs = fp8_ld(m.H);
  up.y = tiles ? hq : b + w.h;
  up.ys = hs;
  up.ld_ys = fp8_ld(m.I);
  up.chunks = gr.chunks;
  up.max_chunks = w.max_chunks;
  up.chunk_rows = w.chunk_rows;
  up.n_chunks = gr.n_chunks;
  up.row_map = gr.row_map;
  up.x_rows = m.T;
  e = fp8_gemm(up, st);
  if (e == hipSuccess && !tiles)
    e = fp8_quantize_rows(b + w.h, true, n, m.I, hq, hs, fp8_ld(m.I), st);
  if (e != hipSuccess) return e;
  down.x = hq;
  down.xs = hs;
  down.ld_xs = fp8_ld(m.I);
  down.y = b + w.y;
  down.out_f32 = 1;
  down.chunks = gr.chunks;
  down.max_chunks = w.max_chunks;
  down.chunk_rows = w.chunk_rows;
  down.n_chunks = gr.n_chunks;
  e = fp8_gemm(down, st);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fp8_combine_kernel, dim3(m.T, (m.H + 1023) / 1024), dim3(256), 0, st,
                     m.residual, reinterpret_cast<const float *>(b + w.y), gr.pos, m.weights, m.H,
                     m.top_k, m.out, m.out_f32);
  return hipGetLastError();
}

}  // namespace cai4
