// tokens.hip -- a layer's slots (token, choice) sorted by expert, rows moved to that
// order and back with the slots' weights, and the gradient of the way back.
//
// Sorting is a counting sort that keeps the slots' order within a group: shares of
// the slots are counted (one launch), then every share adds up the counts before its
// own and places its slots (another); one share does both by itself.  The rank of a
// slot among the slots of its group comes from ballots, not from the order in which
// atomics return, so that the result is the same every time.
//
// The other three move rows and are bound by HBM: a token's row is read once for all
// of its slots.
#include "fp8.hpp"
#include "rows.hpp"
#include "tokens.hpp"

namespace cai4 {
namespace {

// ---- sort ----

constexpr int kSortThreads = 256, kSortWaves = 4;
constexpr int kSortPer = kSortMaxGroups / kSortThreads;  // neighbouring groups per thread
constexpr int kShareSlots = 1024, kMaxShares = 64;
int shares_of(int n) {
  const int s = (n + kShareSlots - 1) / kShareSlots;
  return s < 1 ? 1 : s < kMaxShares ? s : kMaxShares;
}
// Counts of a share: its groups, then the slots left out, in whole 16 bytes.
__host__ __device__ inline int ld_counts(int E) { return (E + 1 + 3) & ~3; }

struct SortLds {
  int cnt[kSortWaves][kSortMaxGroups + 4];  // counts; then next rows
  int waves[kSortWaves];
  int left_out;
};

// A wave's slots of share b: [first, last).
CAI4_DEV void wave_slots(const SortTokens &s, int shares, int b, int wave, int &first, int &last) {
  const int per_wave = ((s.n + shares * kSortWaves - 1) / (shares * kSortWaves) + 63) & ~63;
  const int64_t at = ((int64_t)b * kSortWaves + wave) * per_wave;
  first = at < s.n ? (int)at : s.n;
  last = s.n - first < per_wave ? s.n : first + per_wave;
}

// The group of slot i; E: left out.
CAI4_DEV int group_of(const SortTokens &s, int i) {
  const int e = s.ids[i];
  const bool in = e >= 0 && e < s.E && !(s.weights && s.weights[i] < s.threshold);
  return in ? e : s.E;
}

CAI4_DEV void count_share(const SortTokens &s, int shares, int b, SortLds &l) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int e = threadIdx.x; e <= s.E; e += kSortThreads)
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) l.cnt[w][e] = 0;
  __syncthreads();
  int first, last;
  wave_slots(s, shares, b, wave, first, last);
  for (int i = first + lane; i < last; i += 64) atomicAdd(&l.cnt[wave][group_of(s, i)], 1);
  __syncthreads();
}

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortTokens s, int shares,
                                                                  int *counts) {
  __shared__ SortLds l;
  count_share(s, shares, blockIdx.x, l);
  const int ld = ld_counts(s.E);
  for (int e = threadIdx.x; e < ld; e += kSortThreads) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) c += e <= s.E ? l.cnt[w][e] : 0;
    counts[(size_t)blockIdx.x * ld + e] = c;
  }
}

__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(SortTokens s, int shares,
                                                                  const int *counts) {
  __shared__ SortLds l;
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e0 = threadIdx.x * kSortPer, ld = ld_counts(s.E);
  count_share(s, shares, b, l);
  // this thread's groups over all shares, and over those before this one
  int total[kSortPer] = {}, before[kSortPer] = {};
  if (shares == 1) {
#pragma unroll
    for (int q = 0; q < kSortPer; ++q)
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) total[q] += e0 + q < s.E ? l.cnt[w][e0 + q] : 0;
  } else if (e0 < s.E) {
    static_assert(kSortPer == 4, "one load per share");
    for (int h = 0; h < shares; ++h) {
      const u32x4_t v = *reinterpret_cast<const u32x4_t *>(counts + (size_t)h * ld + e0);
#pragma unroll
      for (int q = 0; q < kSortPer; ++q) {
        const int c = e0 + q < s.E ? (int)v[q] : 0;
        total[q] += c;
        before[q] += h < b ? c : 0;
      }
    }
  }
  int left = 0;  // left out before this share (wave 0: a share per lane)
  if (wave == 0) {
    for (int h = lane; h < b; h += 64) left += counts[(size_t)h * ld + s.E];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) left += __shfl_xor(left, d);
  }
  // first rows: a sum over the threads before this one
  int mine = 0;
#pragma unroll
  for (int q = 0; q < kSortPer; ++q) mine += total[q];
  int row = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(row, d);
    if (lane >= d) row += u;
  }
  if (lane == 63) l.waves[wave] = row;
  if (wave == 0 && lane == 0) l.left_out = left;
  __syncthreads();
  row -= mine;
  for (int w = 0; w < wave; ++w) row += l.waves[w];
#pragma unroll
  for (int q = 0; q < kSortPer; ++q) {
    const int e = e0 + q;
    if (e < s.E) {
      if (b == 0) s.offsets[e] = row;
      int at = row + before[q];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = l.cnt[w][e];
        l.cnt[w][e] = at;
        at += c;
      }
    }
    row += total[q];
  }
  if (threadIdx.x == kSortThreads - 1) {  // (row: all that are kept)
    if (b == 0) s.offsets[s.E] = row;
    int at = row + l.left_out;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = l.cnt[w][s.E];
      l.cnt[w][s.E] = at;
      at += c;
    }
  }
  __syncthreads();
  int first, last;
  wave_slots(s, shares, b, wave, first, last);
  int *next = l.cnt[wave];
  for (int i0 = first; i0 < last; i0 += 64) {
    const int i = i0 + lane;
    const bool here = i < last;
    const int e = here ? group_of(s, i) : 0;
    uint64_t same = __ballot(here);  // the lanes of this one's group
#pragma unroll
    for (int bit = 0; bit < 11; ++bit) {
      const uint64_t on = __ballot((e >> bit) & 1);
      same &= (e >> bit) & 1 ? on : ~on;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (here) {
      const int p = next[e] + rank;
      s.slots[p] = i;
      s.rows[i] = e < s.E ? p : -1;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (one wave's LDS)
    if (here && rank == 0) next[e] += __popcll(same);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- rows ----

constexpr int kMoveThreads = 256;

// A run of a token's row to the rows of its slots.
template <bool FULL, class X, class Y, int V>
CAI4_DEV void gather_run(const X *x, const int32_t *__restrict__ rows, int n, int k, int cols,
                         Y *xs, int left) {
  const Run<X, V> in = load_some<FULL, X, V>(x, left);
  Run<Y, V> out;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (sizeof(X) == sizeof(Y))
      out.v[i] = in.v[i];
    else
      out.v[i] = row_value<Y>(value_of_row(in.v[i]));
  }
  for (int j = 0; j < k; ++j) {
    const int p = rows[j];
    if (p >= 0 && p < n) store_some<FULL, Y, V>(xs + (size_t)p * cols, out, left);
  }
}

template <class X, class Y, int V>
__global__ __launch_bounds__(kMoveThreads) void gather_kernel(const X *x,
                                                              const int32_t *__restrict__ rows,
                                                              int n, int k, int cols, Y *xs) {
  const int t = blockIdx.x, c = (blockIdx.y * kMoveThreads + threadIdx.x) * V;
  const int left = cols - c;
  x += (size_t)t * cols + c;
  rows += (size_t)t * k;
  if (left >= V)
    gather_run<true, X, Y, V>(x, rows, n, k, cols, xs + c, left);
  else if (left > 0)
    gather_run<false, X, Y, V>(x, rows, n, k, cols, xs + c, left);
}

template <bool FULL, class Y, class O, int V>
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
    const Run<Y, V> y = load_some<FULL, Y, V>(ys + (size_t)p * a.cols, left);
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
  store_some<FULL, O, V>(static_cast<O *>(a.out) + o, out, left);
}

template <class Y, class O, int V>
__global__ __launch_bounds__(kMoveThreads) void combine_kernel(CombineTokens a) {
  const int t = blockIdx.x, c = (blockIdx.y * kMoveThreads + threadIdx.x) * V;
  const int left = a.cols - c;
  if (left >= V)
    combine_run<true, Y, O, V>(a, t, c, left);
  else if (left > 0)
    combine_run<false, Y, O, V>(a, t, c, left);
}

constexpr int kGradSlots = 8;  // of one workgroup

template <bool FULL, class D, class Y, int V>
CAI4_DEV void grad_run(const CombineGrad &a, int t, int c, int left, const int (&p)[kGradSlots],
                       const float (&w)[kGradSlots], float (&dot)[kGradSlots]) {
  const Run<D, V> d =
      load_some<FULL, D, V>(static_cast<const D *>(a.dout) + (size_t)t * a.cols + c, left);
#pragma unroll
  for (int j = 0; j < kGradSlots; ++j) {
    if (p[j] < 0) continue;
    const size_t at = (size_t)p[j] * a.cols + c;
    const Run<Y, V> y = load_some<FULL, Y, V>(static_cast<const Y *>(a.ys) + at, left);
    Run<Y, V> g;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float v = value_of_row(d.v[i]);
      dot[j] = __fmaf_rn(v, value_of_row(y.v[i]), dot[j]);
      g.v[i] = row_value<Y>(w[j] * v);
    }
    store_some<FULL, Y, V>(static_cast<Y *>(a.dys) + at, g, left);
  }
}

template <class D, class Y, int V>
__global__ __launch_bounds__(kMoveThreads) void combine_grad_kernel(CombineGrad a) {
  __shared__ float part[kMoveThreads / 64][kGradSlots];
  const int t = blockIdx.x, j0 = blockIdx.y * kGradSlots;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.T * a.top_k;
  int p[kGradSlots];
  float w[kGradSlots], dot[kGradSlots] = {};
#pragma unroll
  for (int j = 0; j < kGradSlots; ++j) {
    const bool in = j0 + j < a.top_k;
    const size_t at = (size_t)t * a.top_k + (in ? j0 + j : 0);
    p[j] = in ? a.rows[at] : -1;
    p[j] = __builtin_amdgcn_readfirstlane(p[j] < n ? p[j] : -1);
    w[j] = a.weights[at];
  }
  int c = threadIdx.x * V;
  for (; c + V <= a.cols; c += kMoveThreads * V)
    grad_run<true, D, Y, V>(a, t, c, V, p, w, dot);
  if (c < a.cols) grad_run<false, D, Y, V>(a, t, c, a.cols - c, p, w, dot);
#pragma unroll
  for (int j = 0; j < kGradSlots; ++j) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) dot[j] += __shfl_xor(dot[j], s);
    if (lane == 0) part[wave][j] = dot[j];
  }
  __syncthreads();
  const int j = threadIdx.x;
  if (j < kGradSlots && j0 + j < a.top_k) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kMoveThreads / 64; ++q) v += part[q][j];
    a.dweights[(size_t)t * a.top_k + j0 + j] = v;
  }
}

dim3 move_grid(int T, int cols, int V) {
  return dim3(T, (cols + kMoveThreads * V - 1) / (kMoveThreads * V));
}

template <class X, class Y>
hipError_t gather(const void *x, const int32_t *rows, int T, int k, int cols, void *xs,
                  hipStream_t st) {
  constexpr int V = 16 / (sizeof(X) > sizeof(Y) ? sizeof(X) : sizeof(Y));
  hipLaunchKernelGGL((gather_kernel<X, Y, V>), move_grid(T, cols, V), dim3(kMoveThreads), 0, st,
                     static_cast<const X *>(x), rows, T * k, k, cols, static_cast<Y *>(xs));
  return hipGetLastError();
}

template <class Y, class O>
hipError_t combine(const CombineTokens &c, hipStream_t st) {
  constexpr int V = 16 / (sizeof(Y) > sizeof(O) ? sizeof(Y) : sizeof(O));
  hipLaunchKernelGGL((combine_kernel<Y, O, V>), move_grid(c.T, c.cols, V), dim3(kMoveThreads), 0,
                     st, c);
  return hipGetLastError();
}

template <class D, class Y>
hipError_t combine_grad(const CombineGrad &c, hipStream_t st) {
  constexpr int V = 16 / (sizeof(D) > sizeof(Y) ? sizeof(D) : sizeof(Y));
  const dim3 grid(c.T, (c.top_k + kGradSlots - 1) / kGradSlots);
  hipLaunchKernelGGL((combine_grad_kernel<D, Y, V>), grid, dim3(kMoveThreads), 0, st, c);
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
    hipLaunchKernelGGL(sort_count_kernel, dim3(shares), dim3(kSortThreads), 0, st, s, shares,
                       counts);
  hipLaunchKernelGGL(sort_place_kernel, dim3(shares), dim3(kSortThreads), 0, st, s, shares,
                     counts);
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
