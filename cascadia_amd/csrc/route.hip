// route.hip -- choice of a layer's experts from its router logits, one wave per
// token.
//
// s = sigmoid(l), or softmax(l) over all experts; c = s + bias.  With groups,
// each group of neighbouring experts is ranked by the sum of its best one or
// two c, and only the experts of the best groups stay.  The top_k by c follow
// (without a bias by l: the same order, and one that no rounding of s blurs),
// ties to the lower id; their weights are s, renormalised and scaled, in 64 bits and
// rounded once (8,192 tokens of 384: 15.5 us; rounded at each step, twice as far off,
// 15.1).
//
// The choice is that of 64-bit scores: a token of some hundred experts has two
// scores next to the border of the chosen ones that 32 bits do not tell apart
// once in some 10^4 tokens, and it would then depend on the rounding of the
// exponential.  It is made from 32-bit scores where all that it rests on lie
// further apart than those can be off (all but one token in some 300), and again
// in 64 bits where they do not.  Lane i holds experts i, i + 64, ...; a round takes
// the wave's maximum and, by ballots in ascending order, the lowest id that has it.
//
// Bound: VALU issue, about 35 instructions a round and token.  8,192 tokens of 384
// experts, top 8 by sigmoid and bias: 16 us, in 64 bits throughout 24.6, which softmax
// scores with a bias take always (333 tokens: 10.1, by sigmoid 10.7).
//
// A NaN logit counts as -infinity.  A softmax whose largest logit is +infinity
// is shared by those that have it; one of a row that is -infinity throughout is
// 0 for every expert.
#include <math.h>

#include "fp8.hpp"
#include "int4_common.hpp"
#include "moe_route.hpp"

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

// Lane k's value (k uniform).
CAI4_DEV double lane_f64(double v, int k) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, k);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), k);
  return __builtin_bit_cast(double, hi << 32 | lo);
}

constexpr int kRouteWaves = 4;

// The choice in 64 bits throughout: chosen id per lane < top_k.
template <int R>
CAI4_DEV int choose64(const RouteExperts &r, const float *logits, double *cs, int lane) {
  const int E = r.E, per = E / r.n_groups;
  double c[R], key[R];
  double mx = -INFINITY, sum = 0.0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 64 * j;
    key[j] = e < E ? (double)logits[e] : -INFINITY;
    mx = fmax(mx, key[j]);
  }
  if (!r.sigmoid) mx = wave_max(mx);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    c[j] = r.sigmoid               ? 1.0 / (1.0 + exp(-key[j]))
           : key[j] == -INFINITY   ? 0.0
           : key[j] == mx          ? 1.0
                                   : exp(key[j] - mx);
    sum += c[j];
  }
  if (!r.sigmoid) {
    sum = wave_sum(sum);
    const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int j = 0; j < R; ++j) c[j] *= inv;
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 64 * j;
    if (r.bias && e < E) c[j] += (double)r.bias[e];
    if (e < E) cs[e] = c[j] != c[j] ? -INFINITY : c[j];
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (one wave's LDS)
  uint64_t kept = ~0ull;
  if (r.n_groups > 1) {
    double gk = -INFINITY;  // this lane's group
    if (lane < r.n_groups) {
      double a = -INFINITY, b = -INFINITY;  // its best two
      for (int i = 0; i < per; ++i) {
        const double v = cs[lane * per + i];
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
    key[j] = in ? key_of(r.bias ? c[j] : key[j]) : -INFINITY;
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
  return id;
}

// What 32-bit scores around v may be off together (each: an exponential, a
// division and a sum of a few steps of 2^-24, scores of at most 1 and their bias).
CAI4_DEV float doubt(float v) { return 0x1p-19f * (1.0f + fabsf(v)); }

// f32 as an integer of the same order (-0 and +0 alike), and back.
CAI4_DEV int order_of(float v) {
  const int b = (int)fbits(v + 0.0f);
  return b ^ ((b >> 31) & 0x7FFFFFFF);
}
CAI4_DEV float value_of(int o) { return bitsf((uint32_t)(o ^ ((o >> 31) & 0x7FFFFFFF))); }
constexpr int kNotThere = (int)0x80000000;  // below order_of(-infinity)

// The largest of a wave's integers, as a scalar: within 16 lanes by DPP, then each
// row of 16 into the next.
CAI4_DEV int wave_max_i32(int v) {
  auto most = [](int a, int b) { return a > b ? a : b; };
  v = most(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true));
  v = most(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true));
  v = most(v, __builtin_amdgcn_mov_dpp(v, 0x124, 0xF, 0xF, true));
  v = most(v, __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true));
  v = most(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));
  v = most(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(v, 63);
}

// The same choice from 32-bit scores; *sure is false (for the whole wave) where two
// of them are too close to say.
template <int R, bool BIAS>
CAI4_DEV int choose32(const RouteExperts &r, const float (&l)[R], const float (&bias)[R], float mx,
                      float *cs, int lane, bool *sure) {
  const int E = r.E;
  int key[R];
  bool ok = true;
  if (BIAS || r.n_groups > 1) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      // (a softmax's common divisor changes no order here: it has no bias)
      const float s = r.sigmoid ? __builtin_amdgcn_rcpf(1.0f + __expf(-l[j])) : __expf(l[j] - mx);
      const float c = BIAS ? s + bias[j] : s;
      if (r.n_groups > 1) cs[lane + 64 * j] = c;
      key[j] = order_of(BIAS ? c : l[j]);
      // a score that is no number (an infinite or NaN bias) is left to 64 bits
      if (BIAS) ok = ok && fabsf(c) < INFINITY;
    }
    if (BIAS) ok = __ballot(!ok) == 0;
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j) key[j] = order_of(l[j]);
  }
  const int per = E / r.n_groups;
  if (r.n_groups > 1) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (one wave's LDS)
    // 2^p lanes per group, joined by swaps; the first of them keeps the group
    int p = 0;
    while ((r.n_groups << (p + 1)) <= 64) ++p;
    const int g = lane >> p;
    float a = -INFINITY, b = -INFINITY;
    if (g < r.n_groups)
      for (int i = lane & ((1 << p) - 1); i < per; i += 1 << p) {
        const float v = cs[g * per + i];
        b = fmaxf(b, fminf(a, v));
        a = fmaxf(a, v);
      }
    for (int d = 1; d < (1 << p); d *= 2) {
      const float a2 = __shfl_xor(a, d), b2 = __shfl_xor(b, d);
      b = fmaxf(fminf(a, a2), fmaxf(b, b2));
      a = fmaxf(a, a2);
    }
    const bool has = g < r.n_groups && !(lane & ((1 << p) - 1));
    // a sum of two is as good as its parts: large ones that cancel are left to 64 bits
    if (BIAS && r.group_best == 2 && per > 1) ok = ok && __ballot(has && b < -1.0f) == 0;
    int gk = has ? order_of(r.group_best == 2 && per > 1 ? a + b : a) : kNotThere;
    uint64_t kept = 0;
    int low = 0;
    for (int i = 0; i < r.top_groups; ++i) {
      low = wave_max_i32(gk);
      const int first = __builtin_ctzll(__ballot(gk == low));
      kept |= 1ull << (first >> p);
      if (lane == first) gk = kNotThere;
    }
    if (r.top_groups < r.n_groups) {
      const float least = value_of(low), next = value_of(wave_max_i32(gk));
      ok = ok && least - next > 2.0f * doubt(least);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int e = lane + 64 * j;
      if (!((kept >> ((e < E ? e : 0) / per)) & 1)) key[j] = kNotThere;
    }
  }
#pragma unroll
  for (int j = 0; j < R; ++j)
    if (lane + 64 * j >= E) key[j] = kNotThere;
  int id = 0, mine = 0;
  const int n = BIAS && r.top_k < r.top_groups * per ? r.top_k + 1 : r.top_k;
  for (int k = 0; k < n; ++k) {
    int m = key[0];
#pragma unroll
    for (int j = 1; j < R; ++j) m = key[j] > m ? key[j] : m;
    m = wave_max_i32(m);
    int first = 0;
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      const uint64_t hit = __ballot(key[j] == m);
      first = hit ? 64 * j + __builtin_ctzll(hit) : first;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) key[j] = lane + 64 * j == first ? kNotThere : key[j];
    const bool here = lane == k;
    id = here ? first : id;
    mine = here ? m : mine;
  }
  // (without a bias the logits themselves are compared: nothing to doubt)
  if (BIAS) {
    const float v = value_of(mine), before = __shfl_up(v, 1);
    ok = ok && __ballot(lane > 0 && lane < n && !(before - v > doubt(v))) == 0;
  }
  *sure = ok;
  return id;
}

template <int R, bool F32, bool BIAS>  // R >= ceil(E / 64): experts per lane, lane + 64 j
__global__ __launch_bounds__(64 * kRouteWaves) void route_experts_kernel(RouteExperts r) {
  __shared__ double cs[kRouteWaves][64 * R];
  __shared__ float ls[kRouteWaves][64 * R];  // logits
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * kRouteWaves + __builtin_amdgcn_readfirstlane(wave);
  if (t >= r.T) return;  // whole waves; no barriers in this kernel
  const int E = r.E;
  float l[R], bias[R], mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < R; ++j) {  // every load first, none behind a branch
    const int e = lane + 64 * j, at = e < E ? e : 0;
    if (F32)
      l[j] = static_cast<const float *>(r.logits)[(size_t)t * E + at];
    else
      l[j] = bf16_to_f32(static_cast<const uint16_t *>(r.logits)[(size_t)t * E + at]);
    bias[j] = BIAS ? r.bias[at] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 64 * j;
    l[j] = l[j] != l[j] || e >= E ? -INFINITY : l[j];
    ls[wave][e] = l[j];
    mx = fmaxf(mx, l[j]);
  }
  double sum = 0.0;
  if (!r.sigmoid) {
    mx = wave_max_f32(mx);
#pragma unroll
    for (int j = 0; j < R; ++j)
      sum += (double)(l[j] == -INFINITY ? 0.f : l[j] == mx ? 1.f : expf(l[j] - mx));
    sum = wave_sum(sum);
  }
  bool sure = false;
  int id = 0;
  // (a softmax's scores are added to a bias in 64 bits only, and where its largest
  // logit is infinite)
  if (r.sigmoid || (!BIAS && fabsf(mx) < INFINITY))
    id = choose32<R, BIAS>(r, l, bias, mx, reinterpret_cast<float *>(cs[wave]), lane, &sure);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (one wave's LDS)
  if (!sure) id = choose64<R>(r, ls[wave], cs[wave], lane);
  // the chosen ones' scores, one per lane
  const double v = lane < r.top_k ? (double)ls[wave][id] : 0.0;
  double s;
  if (r.sigmoid)
    s = 1.0 / (1.0 + exp(-v));
  else
    s = v == -INFINITY ? 0.0 : (v == (double)mx ? 1.0 : exp(v - (double)mx)) / sum;
  if (r.normalize) {
    double total = 0.0;
    for (int k = 0; k < r.top_k; ++k) total += lane_f64(s, k);
    s = s / (total + 1.0e-20);
  }
  if (lane < r.top_k) {
    r.ids[(size_t)t * r.top_k + lane] = id;
    r.weights[(size_t)t * r.top_k + lane] = (float)(s * (double)r.scale);
  }
}

template <int R>
void route_launch(const RouteExperts &r, dim3 grid, dim3 block, hipStream_t st) {
  if (r.x_f32 && r.bias)
    hipLaunchKernelGGL((route_experts_kernel<R, true, true>), grid, block, 0, st, r);
  else if (r.x_f32)
    hipLaunchKernelGGL((route_experts_kernel<R, true, false>), grid, block, 0, st, r);
  else if (r.bias)
    hipLaunchKernelGGL((route_experts_kernel<R, false, true>), grid, block, 0, st, r);
  else
    hipLaunchKernelGGL((route_experts_kernel<R, false, false>), grid, block, 0, st, r);
}

}  // namespace

hipError_t route_experts(const RouteExperts &r, hipStream_t st) {
  const dim3 grid((r.T + kRouteWaves - 1) / kRouteWaves), block(64 * kRouteWaves);
  const int n = (r.E + 63) / 64;
  if (n <= 1)
    route_launch<1>(r, grid, block, st);
  else if (n <= 2)
    route_launch<2>(r, grid, block, st);
  else if (n <= 4)
    route_launch<4>(r, grid, block, st);
  else if (n <= 6)
    route_launch<6>(r, grid, block, st);
  else if (n <= 8)
    route_launch<8>(r, grid, block, st);
  else
    route_launch<16>(r, grid, block, st);
  return hipGetLastError();
}

}  // namespace cai4
