// route.hip -- choice of a layer's experts from its router logits, one wave per
// token.
//
// s = sigmoid(l), or softmax(l) over all experts; c = s + bias.  With groups,
// each group of neighbouring experts is ranked by the sum of its best one or
// two c, and only the experts of the best groups stay.  The top_k by c follow
// (without a bias by l: the same order, and one that no rounding of s blurs),
// ties to the lower id; their weights are s, renormalised and scaled.
//
// Scores are computed and compared in 64 bits: a token of some hundred experts
// has two scores next to the border of the chosen ones that 32 bits do not tell
// apart once in some 10^4 tokens, and the choice would then depend on the
// rounding of the exponential.  Lane i holds experts i, i + 64, ...; a round
// takes the wave's maximum and, by ballots in ascending order, the lowest id
// that has it.
//
// A NaN logit counts as -infinity.  A softmax whose largest logit is +infinity
// is shared by those that have it; one of a row that is -infinity throughout is
// 0 for every expert.
#include <math.h>

#include "fp8.hpp"
#include "int4_common.hpp"

namespace cai4 {
namespace {

// -infinity among the scores (and NaN): below them all, above what is not there.
constexpr double kLeast = -1.0e308;
CAI4_DEV double key_of(double c) { return c > kLeast ? c : kLeast; }

CAI4_DEV double wave_max(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = fmax(v, __shfl_xor(v, d));
  return v;
}
CAI4_DEV double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

constexpr int kRouteWaves = 4;

template <int R>  // R >= ceil(E / 64): experts per lane, lane + 64 j
__global__ __launch_bounds__(64 * kRouteWaves) void route_experts_kernel(RouteExperts r) {
  __shared__ double cs[kRouteWaves][64 * R];  // c of every expert (groups)
  __shared__ float ss[kRouteWaves][64 * R];   // s
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * kRouteWaves + wave;
  const bool live = t < r.T;
  const int E = r.E;
  double l[R], s[R], key[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 64 * j;
    l[j] = -INFINITY;
    if (live && e < E) {
      const size_t at = (size_t)t * E + e;
      const float v = r.x_f32 ? static_cast<const float *>(r.logits)[at]
                              : bf16_to_f32(static_cast<const uint16_t *>(r.logits)[at]);
      l[j] = v != v ? -INFINITY : (double)v;
    }
  }
  if (r.sigmoid) {
#pragma unroll
    for (int j = 0; j < R; ++j) s[j] = 1.0 / (1.0 + exp(-l[j]));
  } else {
    double mx = -INFINITY, sum = 0.0;
#pragma unroll
    for (int j = 0; j < R; ++j) mx = fmax(mx, l[j]);
    mx = wave_max(mx);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      s[j] = l[j] == -INFINITY ? 0.0 : l[j] == mx ? 1.0 : exp(l[j] - mx);
      sum += s[j];
    }
    sum = wave_sum(sum);
    const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int j = 0; j < R; ++j) s[j] *= inv;
  }
  double c[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 64 * j;
    c[j] = s[j] + (r.bias && e < E ? (double)r.bias[e] : 0.0);
    ss[wave][e] = (float)s[j];
    if (r.n_groups > 1) cs[wave][e] = c[j] != c[j] ? -INFINITY : c[j];
  }
  __syncthreads();
  uint64_t kept = ~0ull;
  const int per = E / r.n_groups;
  if (r.n_groups > 1) {
    double gk = -INFINITY;  // this lane's group
    if (lane < r.n_groups) {
      double a = -INFINITY, b = -INFINITY;  // its best two
      for (int i = 0; i < per; ++i) {
        const double v = cs[wave][lane * per + i];
        b = fmax(b, fmin(a, v));
        a = fmax(a, v);
      }
      gk = key_of(r.group_best == 2 && per > 1 ? a + b : a);
    }
    kept = 0;
    for (int i = 0; i < r.top_groups; ++i) {
      const double m = wave_max(gk);
      const int first = __builtin_ctzll(__ballot(gk == m));
      kept |= 1ull << first;
      if (lane == first) gk = -INFINITY;
    }
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 64 * j;
    const bool in = e < E && (r.n_groups == 1 || ((kept >> (e / per)) & 1));
    key[j] = in ? key_of(r.bias ? c[j] : l[j]) : -INFINITY;
  }
  int id = 0;
  for (int k = 0; k < r.top_k; ++k) {
    double m = key[0];
#pragma unroll
    for (int j = 1; j < R; ++j) m = fmax(m, key[j]);
    m = wave_max(m);
    int first = -1;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const uint64_t hit = __ballot(key[j] == m);
      const bool mine = first < 0 && hit;
      first = mine ? 64 * j + __builtin_ctzll(hit) : first;
      key[j] = mine && lane == (first & 63) ? -INFINITY : key[j];
    }
    if (lane == k) id = first;
  }
  float w = lane < r.top_k ? ss[wave][id] : 0.f;
  if (r.normalize) {
    float sum = 0.f;
    for (int k = 0; k < r.top_k; ++k) sum += __shfl(w, k);
    w = w / (sum + 1.0e-20f);
  }
  if (live && lane < r.top_k) {
    r.ids[(size_t)t * r.top_k + lane] = id;
    r.weights[(size_t)t * r.top_k + lane] = w * r.scale;
  }
}

}  // namespace

hipError_t route_experts(const RouteExperts &r, hipStream_t st) {
  const dim3 grid((r.T + kRouteWaves - 1) / kRouteWaves), block(64 * kRouteWaves);
  const int n = (r.E + 63) / 64;
  if (n <= 1)
    hipLaunchKernelGGL(route_experts_kernel<1>, grid, block, 0, st, r);
  else if (n <= 2)
    hipLaunchKernelGGL(route_experts_kernel<2>, grid, block, 0, st, r);
  else if (n <= 4)
    hipLaunchKernelGGL(route_experts_kernel<4>, grid, block, 0, st, r);
  else if (n <= 8)
    hipLaunchKernelGGL(route_experts_kernel<8>, grid, block, 0, st, r);
  else
    hipLaunchKernelGGL(route_experts_kernel<16>, grid, block, 0, st, r);
  return hipGetLastError();
}

}  // namespace cai4
