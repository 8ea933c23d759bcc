// tokens.hip -- a layer's slots (token, choice) sorted by expert, rows moved to that
// order and back with the slots' weights, and the gradient of the way back.
//
// Sorting is a counting sort that keeps the slots' order within a group: row of slot i =
// slots of smaller groups + slots before i of its own.  Shares of the slots are counted
// (one launch), then every share adds up the counts before its own and places its slots
// (another); up to 4,096 slots are one share, which does both by itself.  A slot's rank
// among the 64 of a wave comes from ballots, not from the order in which atomics
// return, so that the result is the same every time.  Bound: launches and a handful of
// dependent loads (12 bytes a slot).  8,192 x 8 slots over 384 experts: 4.2 + 9 us.
//
// The other three move rows and are bound by HBM:
//   gather   xs[row(t, j)] = x[t]            a token's row read once for its slots
//   combine  out[t] = res[t] + sum w y       each slot's row read once
//   gradient dy[row] = w dout, dw = y . dout  both in one pass over y
// 4,096 tokens, 8 slots each, rows of 7,168 in bf16: gather 88 us (514 MB, 5.8 TB/s),
// combine 111 (574 MB, 5.2); the gradient of rows of 4,096: 104 us (555 MB, 5.3).  A copy
// of 2 GiB reaches 4.9: these write and read past the caches (below).
#include "fp8.hpp"
#include "rows.hpp"
#include "tokens.hpp"

namespace cai4 {
namespace {

// ---- sort ----

// Each wave of a workgroup places a run of neighbouring slots; its threads share the
// groups among them.  Sixteen waves, or four for up to 1,024 slots (128 slots of 256
// experts: the kernel takes 4.6 us, with sixteen 5.3).
constexpr int kSortWaves = 16, kFewWaves = 4;
constexpr int kSteps = 4;  // steps of 64 slots whose ids are loaded together
// Slots of a share, so that each wave takes one load of ids; at most 128 shares (a
// placing workgroup adds up the counts of all shares).
constexpr int kShareSlots = kSortWaves * kSteps * 64, kMaxShares = 128;
constexpr int kFewSlots = kFewWaves * kSteps * 64;
int shares_of(int n) {
  const int s = (n + kShareSlots - 1) / kShareSlots;
  return s < 1 ? 1 : s < kMaxShares ? s : kMaxShares;
}
// Counts of a share: its groups, then the slots left out.
__host__ __device__ inline int ld_counts(int E) { return E + 1; }

// A wave's slots of share b: [first, last).
template <int W>
CAI4_DEV void wave_slots(const SortTokens &s, int shares, int b, int wave, int &first, int &last) {
  const int waves = shares * W;
  const int per = ((s.n + waves - 1) / waves + 63) & ~63;
  const int64_t at = ((int64_t)b * W + wave) * per;
  first = at < s.n ? (int)at : s.n;
  last = s.n - first < per ? s.n : first + per;
}

// The groups of slots at + 64 i + lane (E: left out; -1: none).
CAI4_DEV void groups_of(const SortTokens &s, int at, int last, int (&e)[kSteps]) {
  const int lane = threadIdx.x & 63;
  int id[kSteps];
  float w[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int k = at + i * 64 + lane;
    id[i] = s.ids[k < last ? k : last - 1];
    w[i] = s.weights ? s.weights[k < last ? k : last - 1] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const bool in = id[i] >= 0 && id[i] < s.E && !(s.weights && w[i] < s.threshold);
    e[i] = at + i * 64 + lane >= last ? -1 : in ? id[i] : s.E;
  }
}

// The lanes of this lane's group e (-1: none), in `bits` ballots.
CAI4_DEV uint64_t lanes_of(int e, int bits) {
  uint64_t same = __ballot(e >= 0);
  for (int bit = 0; bit < bits; ++bit) {
    const uint64_t mine = (e >> bit) & 1 ? ~0ull : 0;
    same &= ~(__ballot(mine != 0) ^ mine);
  }
  return same;
}

// The places of a wave's next 64 slots behind next[] of their groups, which moves on.
CAI4_DEV int take_places(int e, int bits, int *next) {
  const uint64_t same = lanes_of(e, bits);
  const int rank = __popcll(same & ((1ull << (threadIdx.x & 63)) - 1));
  const int at = e >= 0 ? next[e] : 0;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (one wave's LDS)
  if (e >= 0 && rank == 0) next[e] = at + __popcll(same);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  return at + rank;
}

__global__ __launch_bounds__(64 * kSortWaves) void sort_count_kernel(SortTokens s, int shares,
                                                                     int *counts) {
  __shared__ int cnt[kSortMaxGroups + 1];
  const int b = blockIdx.x, ld = ld_counts(s.E);
  for (int e = threadIdx.x; e <= s.E; e += 64 * kSortWaves) cnt[e] = 0;
  __syncthreads();
  int first, last, e[kSteps];
  wave_slots<kSortWaves>(s, shares, b, threadIdx.x >> 6, first, last);
  for (int at = first; at < last; at += kSteps * 64) {
    groups_of(s, at, last, e);
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      if (e[i] >= 0) atomicAdd(&cnt[e[i]], 1);  // (sums: in any order)
  }
  __syncthreads();
  for (int i = threadIdx.x; i <= s.E; i += 64 * kSortWaves) counts[(size_t)b * ld + i] = cnt[i];
}

template <int W>
__global__ __launch_bounds__(64 * W) void sort_place_kernel(SortTokens s, int shares,
                                                            const int *counts) {
  constexpr int kThreads = 64 * W, kPer = kSortMaxGroups / kThreads;  // groups of a thread
  __shared__ int cnt[W][kSortMaxGroups + 1];  // counts; then next rows
  __shared__ int sums[W + 1];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e0 = threadIdx.x * kPer, ld = ld_counts(s.E);
  const int bits = 32 - __builtin_clz(s.E);
  int first, last, e[kSteps], place[kSteps];
  wave_slots<W>(s, shares, b, wave, first, last);
  if (first < last) groups_of(s, first, last, e);
  // the counts of the first shares, on their way while this one's slots are counted
  constexpr int kLoads = 16;
  const bool many = W == kSortWaves && shares > 1;
  const int *const mine_of = counts + (e0 < s.E ? e0 : s.E);
  int v[kLoads] = {};
  if (many)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = mine_of[(size_t)(i < shares ? i : 0) * ld];
  for (int i = threadIdx.x; i <= s.E; i += kThreads)
#pragma unroll
    for (int w = 0; w < W; ++w) cnt[w][i] = 0;
  __syncthreads();
  for (int at = first; at < last; at += kSteps * 64) {
    if (at > first) groups_of(s, at, last, e);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) place[i] = take_places(e[i], bits, cnt[wave]);
  }
  // the groups' slots over all shares, and over those before this one
  int total[kPer] = {}, before[kPer] = {}, left = 0;
  if (many) {
    static_assert(kSortMaxGroups == 64 * kSortWaves, "a group per thread");
    for (int h0 = 0; h0 < shares; h0 += kLoads) {
      if (h0 > 0)
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          v[i] = mine_of[(size_t)(h0 + i < shares ? h0 + i : h0) * ld];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        total[0] += h0 + i < shares ? v[i] : 0;
        before[0] += h0 + i < b ? v[i] : 0;
      }
    }
    if (wave == 0) {  // slots left out before this share: a share per lane
      for (int h = lane; h < b; h += 64) left += counts[(size_t)h * ld + s.E];
#pragma unroll
      for (int d = 1; d < 64; d *= 2) left += __shfl_xor(left, d);
    }
  }
  __syncthreads();
  int c[kPer][W], mine = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const bool in = e0 + q < s.E;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      c[q][w] = in ? cnt[w][e0 + q] : 0;
      if (shares == 1) total[q] += c[q][w];
    }
    if (!in) total[q] = 0;
    mine += total[q];
  }
  // first rows: a sum over the threads before this one
  int row = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(row, d);
    if (lane >= d) row += u;
  }
  if (lane == 63) sums[wave] = row;
  if (threadIdx.x == 0) sums[W] = left;
  __syncthreads();
  row -= mine;
#pragma unroll
  for (int w = 0; w < W; ++w) row += w < wave ? sums[w] : 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    if (e0 + q < s.E) {
      if (b == 0) s.offsets[e0 + q] = row;
      int at = row + before[q];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        cnt[w][e0 + q] = at;
        at += c[q][w];
      }
    }
    row += total[q];
  }
  if (threadIdx.x == kThreads - 1) {  // (row: all that are kept)
    if (b == 0) s.offsets[s.E] = row;
    int at = row + sums[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int n = cnt[w][s.E];
      cnt[w][s.E] = at;
      at += n;
    }
  }
  __syncthreads();
  // a wave's only ids and their places are still there; of several loads of them they are
  // found again
  int *next = cnt[wave];
  const bool once = first + kSteps * 64 >= last;
  for (int at = first; at < last; at += kSteps * 64) {
    if (!once) groups_of(s, at, last, e);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int p = once ? (e[i] >= 0 ? next[e[i]] : 0) + place[i] : take_places(e[i], bits, next);
      // (p is out of range only where ids or the counts changed meanwhile: another call over
      // the same workspace)
      if (e[i] < 0 || (uint32_t)p >= (uint32_t)s.n) continue;
      const int k = at + i * 64 + lane;
      s.slots[p] = k;
      s.rows[k] = e[i] < s.E ? p : -1;
    }
  }
}

// ---- rows ----

constexpr int kMoveThreads = 256;

constexpr int kBatch = 8;  // slots whose row numbers are loaded together

// The rows of slots j0 .. j0 + B of a token; -1: left out or not there.
template <int B>
CAI4_DEV void rows_of(const int32_t *__restrict__ rows, int n, int k, int t, int j0, int (&p)[B]) {
#pragma unroll
  for (int j = 0; j < B; ++j) {
    p[j] = rows[(size_t)t * k + (j0 + j < k ? j0 + j : 0)];
    p[j] = __builtin_amdgcn_readfirstlane(j0 + j < k && p[j] < n ? p[j] : -1);
  }
}

// A run of a token's row to the rows of its slots.
template <bool FULL, bool STREAM, class X, class Y, int V>
CAI4_DEV void gather_run(const X *x, const int32_t *__restrict__ rows, int n, int k, int t,
                         int cols, Y *xs, int left) {
  const Run<X, V> in = load_some<FULL, X, V>(x, left);
  Run<Y, V> out;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (sizeof(X) == sizeof(Y))
      out.v[i] = in.v[i];
    else
      out.v[i] = row_value<Y>(value_of_row(in.v[i]));
  }
  for (int j0 = 0; j0 < k; j0 += kBatch) {
    int p[kBatch];
    rows_of(rows, n, k, t, j0, p);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (p[j] >= 0) store_some<FULL, STREAM>(xs + (size_t)p[j] * cols, out, left);
  }
}

template <bool STREAM, class X, class Y, int V>
__global__ __launch_bounds__(kMoveThreads) void gather_kernel(const X *x,
                                                              const int32_t *__restrict__ rows,
                                                              int n, int k, int cols, Y *xs) {
  const int t = blockIdx.x, c = (blockIdx.y * kMoveThreads + threadIdx.x) * V;
  const int left = cols - c;
  x += (size_t)t * cols + c;
  if (left >= V)
    gather_run<true, STREAM, X, Y, V>(x, rows, n, k, t, cols, xs + c, left);
  else if (left > 0)
    gather_run<false, STREAM, X, Y, V>(x, rows, n, k, t, cols, xs + c, left);
}

// (Slot by slot: many waves, rather than many loads of a wave, keep HBM busy.)
template <bool FULL, bool STREAM, class Y, class O, int V>
CAI4_DEV void combine_run(const CombineTokens &a, int t, int c, int left) {
  const int n = a.T * a.top_k;
  const Y *ys = static_cast<const Y *>(a.ys) + c;
  const int32_t *__restrict__ rows = a.rows + (size_t)t * a.top_k;
  const float *__restrict__ weights = a.weights ? a.weights + (size_t)t * a.top_k : nullptr;
  float sum[V] = {};
  for (int j = 0; j < a.top_k; ++j) {
    const int p = rows[j];
    if (p < 0 || p >= n) continue;
    const float w = weights ? weights[j] : 1.0f;
    const Run<Y, V> y = load_some<FULL, Y, V, STREAM>(ys + (size_t)p * a.cols, left);
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = __fmaf_rn(w, value_of_row(y.v[i]), sum[i]);
  }
  const size_t o = (size_t)t * a.cols + c;
  if (a.residual) {
    const Run<O, V> r = load_some<FULL, O, V>(static_cast<const O *>(a.residual) + o, left);
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = value_of_row(r.v[i]) + sum[i];
  }
  Run<O, V> out;
#pragma unroll
  for (int i = 0; i < V; ++i) out.v[i] = row_value<O>(sum[i]);
  store_some<FULL>(static_cast<O *>(a.out) + o, out, left);
}

template <bool STREAM, class Y, class O, int V>
__global__ __launch_bounds__(kMoveThreads) void combine_kernel(CombineTokens a) {
  const int t = blockIdx.x, c = (blockIdx.y * kMoveThreads + threadIdx.x) * V;
  const int left = a.cols - c;
  if (left >= V)
    combine_run<true, STREAM, Y, O, V>(a, t, c, left);
  else if (left > 0)
    combine_run<false, STREAM, Y, O, V>(a, t, c, left);
}

// Slots of a workgroup of the gradient: dout is read again for every two, from the
// L2; 4,096 tokens x 8 x 4,096 in bf16: 8 slots 107 us, 4 103.8, 2 104.2, 1 113; 77 x 6 x
// 3,584 in f32: 9.9, 9.0, 8.3, 8.3.
constexpr int kGradThreads = 256, kGradBatch = 2;

template <bool FULL, bool STREAM, class D, class Y, int V>
CAI4_DEV void grad_run(const CombineGrad &a, int t, int c, int left, const int (&p)[kGradBatch],
                       const float (&w)[kGradBatch], float (&dot)[kGradBatch]) {
  const Run<D, V> d =
      load_some<FULL, D, V>(static_cast<const D *>(a.dout) + (size_t)t * a.cols + c, left);
  Run<Y, V> y[kGradBatch];
#pragma unroll
  for (int j = 0; j < kGradBatch; ++j)  // every load before the first use
    if (p[j] >= 0)
      y[j] = load_some<FULL, Y, V, STREAM>(
          static_cast<const Y *>(a.ys) + (size_t)p[j] * a.cols + c, left);
#pragma unroll
  for (int j = 0; j < kGradBatch; ++j) {
    if (p[j] < 0) continue;
    Run<Y, V> g;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float v = value_of_row(d.v[i]);
      dot[j] = __fmaf_rn(v, value_of_row(y[j].v[i]), dot[j]);
      g.v[i] = row_value<Y>(w[j] * v);
    }
    store_some<FULL, STREAM>(static_cast<Y *>(a.dys) + (size_t)p[j] * a.cols + c, g, left);
  }
}

template <bool STREAM, class D, class Y, int V>
__global__ __launch_bounds__(kGradThreads) void combine_grad_kernel(CombineGrad a) {
  __shared__ float part[kGradThreads / 64][kGradBatch];
  const int t = blockIdx.x, j0 = blockIdx.y * kGradBatch;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int p[kGradBatch];
  float w[kGradBatch], dot[kGradBatch] = {};
  rows_of(a.rows, a.T * a.top_k, a.top_k, t, j0, p);
#pragma unroll
  for (int j = 0; j < kGradBatch; ++j)
    w[j] = a.weights[(size_t)t * a.top_k + (j0 + j < a.top_k ? j0 + j : 0)];
  int c = threadIdx.x * V;
  for (; c + V <= a.cols; c += kGradThreads * V)
    grad_run<true, STREAM, D, Y, V>(a, t, c, V, p, w, dot);
  if (c < a.cols) grad_run<false, STREAM, D, Y, V>(a, t, c, a.cols - c, p, w, dot);
#pragma unroll
  for (int j = 0; j < kGradBatch; ++j) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) dot[j] += __shfl_xor(dot[j], s);
    if (lane == 0) part[wave][j] = dot[j];
  }
  __syncthreads();
  const int j = threadIdx.x;
  if (j < kGradBatch && j0 + j < a.top_k) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kGradThreads / 64; ++q) v += part[q][j];
    a.dweights[(size_t)t * a.top_k + j0 + j] = v;
  }
}

dim3 move_grid(int T, int cols, int V) {
  return dim3(T, (cols + kMoveThreads * V - 1) / (kMoveThreads * V));
}

// Whether the slots' rows are written or read past the caches' replacement: more of them
// than the Infinity Cache (256 MiB) holds, in whole lines.  Gather, written so or not:
// 470 MB 89 / 106 us, 134 MB 26.2 / 26.9, 67 MB 12.7 / 12.6; combine, read so or not
// (residual and output in that cache): 470 MB 97 / 119, 101 MB 29.3 / 22.2 (then the rows
// are in it as well); the gradient, both: 268 MB 104 /
// 114; rows of an odd number of bytes, written so: 37 / 31.
constexpr size_t kStreamBytes = (size_t)256 << 20, kLine = 128;
bool streams(const void *p, int rows, int cols, size_t size) {
  return (size_t)rows * cols * size >= kStreamBytes && cols * size % kLine == 0 &&
         (uintptr_t)p % kLine == 0;
}

template <class X, class Y>
hipError_t gather(const void *x, const int32_t *rows, int T, int k, int cols, void *xs,
                  hipStream_t st) {
  constexpr int V = 16 / (sizeof(X) > sizeof(Y) ? sizeof(X) : sizeof(Y));
  const dim3 grid = move_grid(T, cols, V), block(kMoveThreads);
  const X *from = static_cast<const X *>(x);
  Y *to = static_cast<Y *>(xs);
  if (streams(xs, T * k, cols, sizeof(Y)))
    hipLaunchKernelGGL((gather_kernel<true, X, Y, V>), grid, block, 0, st, from, rows, T * k, k,
                       cols, to);
  else
    hipLaunchKernelGGL((gather_kernel<false, X, Y, V>), grid, block, 0, st, from, rows, T * k, k,
                       cols, to);
  return hipGetLastError();
}

template <class Y, class O>
hipError_t combine(const CombineTokens &c, hipStream_t st) {
  constexpr int V = 16 / (sizeof(Y) > sizeof(O) ? sizeof(Y) : sizeof(O));
  const dim3 grid = move_grid(c.T, c.cols, V), block(kMoveThreads);
  if (streams(c.ys, c.T * c.top_k, c.cols, sizeof(Y)))
    hipLaunchKernelGGL((combine_kernel<true, Y, O, V>), grid, block, 0, st, c);
  else
    hipLaunchKernelGGL((combine_kernel<false, Y, O, V>), grid, block, 0, st, c);
  return hipGetLastError();
}

template <class D, class Y>
hipError_t combine_grad(const CombineGrad &c, hipStream_t st) {
  constexpr int V = 16 / (sizeof(D) > sizeof(Y) ? sizeof(D) : sizeof(Y));
  const dim3 grid(c.T, (c.top_k + kGradBatch - 1) / kGradBatch), block(kGradThreads);
  if (streams(c.dys, c.T * c.top_k, c.cols, sizeof(Y)))
    hipLaunchKernelGGL((combine_grad_kernel<true, D, Y, V>), grid, block, 0, st, c);
  else
    hipLaunchKernelGGL((combine_grad_kernel<false, D, Y, V>), grid, block, 0, st, c);
  return hipGetLastError();
}

}  // namespace

size_t sort_tokens_workspace(int n, int E) {
  const int s = shares_of(n);
  return s == 1 ? 0 : (size_t)s * ld_counts(E) * 4;
}

hipError_t sort_tokens(const SortTokens &s, void *workspace, hipStream_t st) {
  const int shares = shares_of(s.n);
  int *counts = static_cast<int *>(workspace);
  if (shares > 1)
    hipLaunchKernelGGL(sort_count_kernel, dim3(shares), dim3(64 * kSortWaves), 0, st, s, shares,
                       counts);
  if (s.n <= kFewSlots)
    hipLaunchKernelGGL(sort_place_kernel<kFewWaves>, dim3(1), dim3(64 * kFewWaves), 0, st, s, 1,
                       counts);
  else
    hipLaunchKernelGGL(sort_place_kernel<kSortWaves>, dim3(shares), dim3(64 * kSortWaves), 0, st, s,
                       shares, counts);
  return hipGetLastError();
}

hipError_t gather_tokens(const void *x, RowType x_type, const int32_t *rows, int T, int top_k,
                         int cols, void *xs, RowType xs_type, hipStream_t st) {
  if (x_type == kRowByte) return gather<uint8_t, uint8_t>(x, rows, T, top_k, cols, xs, st);
  if (x_type == kRowF32)
    return xs_type == kRowF32 ? gather<float, float>(x, rows, T, top_k, cols, xs, st)
                              : gather<float, uint16_t>(x, rows, T, top_k, cols, xs, st);
  return xs_type == kRowF32 ? gather<uint16_t, float>(x, rows, T, top_k, cols, xs, st)
                            : gather<uint16_t, uint16_t>(x, rows, T, top_k, cols, xs, st);
}

hipError_t combine_tokens(const CombineTokens &c, hipStream_t st) {
  if (c.y_f32)
    return c.out_f32 ? combine<float, float>(c, st) : combine<float, uint16_t>(c, st);
  return c.out_f32 ? combine<uint16_t, float>(c, st) : combine<uint16_t, uint16_t>(c, st);
}

hipError_t combine_tokens_grad(const CombineGrad &c, hipStream_t st) {
  if (c.dout_f32)
    return c.y_f32 ? combine_grad<float, float>(c, st) : combine_grad<float, uint16_t>(c, st);
  return c.y_f32 ? combine_grad<uint16_t, float>(c, st)
                 : combine_grad<uint16_t, uint16_t>(c, st);
}

}  // namespace cai4
