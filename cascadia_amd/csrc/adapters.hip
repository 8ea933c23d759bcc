// adapters.hip -- low-rank adapters of many requests at once:
//   y_t = base_t + s_a B_a (A_a x_t),  a: row t's adapter (rows without one: base_t)
//
// Rows come sorted by adapter, in chunks of up to kChunkRows rows of one adapter.
// Two launches: u = A x for every chunk (K in slices where chunks are few; their
// partial sums stay f32), then y = base + B (s u), which adds the slices in order.
//
// Both products run on bf16 MFMAs with f32 sums.  A and B are bf16; f32 x, and u,
// enter as a sum of bf16 planes, each the rounding of what the ones before left
// over: three hold 24 bits, two (for bf16 y) 16.
#include <type_traits>

#include "adapters_common.hpp"
#include "rows.hpp"
#include "tokens.hpp"

namespace cai4 {
namespace {

constexpr int kTiles = kChunkRows / 16;

// v as N bf16 planes whose sum holds 8 N bits of it.  An infinity or NaN is in the
// first alone: what it leaves over would be NaN.
template <int N>
CAI4_DEV void planes_of(float v, uint32_t (&p)[N]) {
  p[0] = split_hi(v);
  float rest = v - bitsf(p[0] << 16);
  if (!(fabsf(v) < INFINITY)) {
    p[0] = f32_to_bf16_rne(v);
    rest = 0.f;
  }
#pragma unroll
  for (int i = 1; i < N; ++i) {
    p[i] = f32_to_bf16_rne(rest);
    rest -= bitsf(p[i] << 16);
  }
}

// Eight values as the operands of N MFMAs.
template <int N>
CAI4_DEV void operands_of(const float (&v)[8], u32x4_t (&op)[N]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo[N], hi[N];
    planes_of<N>(v[2 * i], lo);
    planes_of<N>(v[2 * i + 1], hi);
#pragma unroll
    for (int p = 0; p < N; ++p) op[p][i] = lo[p] | hi[p] << 16;
  }
}

// ---- u = A x ----

constexpr int kRankTile = 64;  // ranks of a workgroup

template <bool F32>
__global__ __launch_bounds__(256) void adapters_in_kernel(Adapters a, float *u, int slices) {
  constexpr int P = F32 ? 3 : 1, RT = kRankTile / 16;
  __shared__ f32x4_t part[4][RT * kTiles][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, q = lane >> 4;
  const Chunk ch = find_chunk(a, blockIdx.x, false);
  if (ch.rows == 0) return;
  const int rank = rank_of(a, ch.group), r0 = blockIdx.z * kRankTile;
  if (r0 >= rank) return;
  const int slice = blockIdx.y;
  // blocks of 128 columns; a wave's are neighbours
  const int blocks = (a.K + 127) / 128, parts = slices * 4, me = slice * 4 + wave;
  const int b0 = (int)((int64_t)blocks * me / parts), b1 = (int)((int64_t)blocks * (me + 1) / parts);
  const uint16_t *A[RT];
  bool a_in[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = r0 + i * 16 + c;
    a_in[i] = r < rank;
    A[i] = a.a + ((size_t)ch.group * a.R + (a_in[i] ? r : 0)) * a.K;
  }
  size_t xo[kTiles];
  bool x_in[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int t = row_of(a, ch, i * 16 + c);
    x_in[i] = t >= 0;
    xo[i] = (size_t)(t < 0 ? 0 : t) * a.ldx;
  }
  f32x4_t acc[RT][kTiles] = {};
  for (int b = b0; b < b1; ++b) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int col = b * 128 + q * 32 + s * 8;
      const bool in = col < a.K;
      u32x4_t av[RT] = {}, xv[kTiles][P] = {};
#pragma unroll
      for (int i = 0; i < RT; ++i)
        if (in && a_in[i]) av[i] = *reinterpret_cast<const u32x4_t *>(A[i] + col);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        if (!(in && x_in[i])) continue;
        if constexpr (F32) {
          const float *p = static_cast<const float *>(a.x) + xo[i] + col;
          const Run<float, 4> lo = load_run<float, 4>(p), hi = load_run<float, 4>(p + 4);
          const float v[8] = {lo.v[0], lo.v[1], lo.v[2], lo.v[3],
                              hi.v[0], hi.v[1], hi.v[2], hi.v[3]};
          operands_of<P>(v, xv[i]);
        } else {
          const Run<uint16_t, 8> v =
              load_run<uint16_t, 8>(static_cast<const uint16_t *>(a.x) + xo[i] + col);
          xv[i][0] = __builtin_bit_cast(u32x4_t, v);
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int p = 0; p < P; ++p) acc[i][j] = mfma_bf16(av[i], xv[j][p], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) part[wave][i * kTiles + j][lane] = acc[i][j];
  __syncthreads();
  // tile i, j: lane holds ranks r0 + 16 i + 4 q + [0, 4) of row 16 j + c
  for (int k = wave; k < RT * kTiles; k += 4) {
    const int i = k / kTiles, j = k % kTiles;
    f32x4_t v = part[0][k][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += part[w][k][lane];
    const int r = r0 + i * 16 + q * 4, row = j * 16 + c;
    if (r < a.R && row < ch.rows)
      *reinterpret_cast<f32x4_t *>(u + ((size_t)slice * a.T + ch.row0 + row) * a.R + r) = v;
  }
}

// ---- y = base + B (s u) ----

constexpr int kColBlock = 64;  // columns of a wave at a time

// What a lane adds to or writes of a row: 16 neighbouring columns.
CAI4_DEV void load16(const void *p, bool f32, size_t at, int left, float (&v)[16]) {
  if (f32) {
    const float *s = static_cast<const float *>(p) + at;
    if (left >= 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Run<float, 4> r = load_run<float, 4>(s + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = r.v[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i < left ? s[i] : 0.f;
    }
  } else {
    const uint16_t *s = static_cast<const uint16_t *>(p) + at;
    if (left >= 16) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Run<uint16_t, 8> r = load_run<uint16_t, 8>(s + 8 * i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * i + j] = bf16_to_f32(r.v[j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i < left ? bf16_to_f32(s[i]) : 0.f;
    }
  }
}
template <bool F32>
CAI4_DEV void store16(void *p, size_t at, int left, const float (&v)[16]) {
  typedef typename std::conditional<F32, float, uint16_t>::type T;
  constexpr int V = 16 / sizeof(T);
  T *d = static_cast<T *>(p) + at;
#pragma unroll
  for (int i = 0; i < 16 / V; ++i) {
    Run<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = row_value<T>(v[V * i + j]);
    if (left >= 16)
      store_run<T, V>(d + V * i, r);
    else
      store_part<T, V>(d + V * i, r, left - V * i);
  }
}

template <bool F32>
__global__ __launch_bounds__(256) void adapters_out_kernel(Adapters a, const float *u, int slices,
                                                           int cols, int bare) {
  constexpr int P = F32 ? 3 : 2;
  extern __shared__ u32x4_t us[];  // [steps of 32 ranks][planes][tiles][lane]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, q = lane >> 4;
  const Chunk ch = find_chunk(a, blockIdx.x, bare);
  if (ch.rows == 0) return;
  const bool own = ch.group < a.E;
  const int rank = own ? rank_of(a, ch.group) : 0, steps = (rank + 31) / 32;
  if (steps) {
    const float s = a.scales ? a.scales[ch.group] : 1.0f;
    for (int k = wave; k < steps * kTiles; k += 4) {
      const int step = k / kTiles, j = k % kTiles;
      const int r = step * 32 + q * 8, row = j * 16 + c;
      float v[8] = {};
      if (row < ch.rows && r < rank) {
        for (int h = 0; h < slices; ++h) {
          const f32x4_t *p = reinterpret_cast<const f32x4_t *>(
              u + ((size_t)h * a.T + ch.row0 + row) * a.R + r);
          const f32x4_t lo = p[0], hi = p[1];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] += lo[i];
            v[4 + i] += hi[i];
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = r + i < rank ? v[i] * s : 0.f;
      }
      u32x4_t op[P];
      operands_of<P>(v, op);
#pragma unroll
      for (int p = 0; p < P; ++p) us[((step * P + p) * kTiles + j) * 64 + lane] = op[p];
    }
    __syncthreads();
  }
  int row[kTiles];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) row[j] = row_of(a, ch, j * 16 + c);
  const uint16_t *B = a.b + (size_t)(own ? ch.group : 0) * a.N * a.R;
  const int n_end = (blockIdx.y + 1) * cols < a.N ? (blockIdx.y + 1) * cols : a.N;
  for (int n0 = blockIdx.y * cols + wave * kColBlock; n0 < n_end; n0 += 4 * kColBlock) {
    f32x4_t acc[4][kTiles] = {};
    for (int step = 0; step < steps; ++step) {
      u32x4_t bv[4];
      const int r = step * 32 + q * 8;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        // (tile m's row i is column 16 (i / 4) + 4 m + i % 4: a lane's outputs are
        // neighbours)
        const int n = n0 + (c >> 2) * 16 + m * 4 + (c & 3);
        bv[m] = u32x4_t{0, 0, 0, 0};
        if (n < a.N && r < rank) {
          bv[m] = *reinterpret_cast<const u32x4_t *>(B + (size_t)n * a.R + r);
          if (r + 8 > rank)  // columns past the rank may hold anything
#pragma unroll
            for (int i = 0; i < 4; ++i)
              bv[m][i] &= (r + 2 * i < rank ? 0xFFFFu : 0u) | (r + 2 * i + 1 < rank ? 0xFFFF0000u : 0u);
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          const u32x4_t uv = us[((step * P + p) * kTiles + j) * 64 + lane];
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[m][j] = mfma_bf16(bv[m], uv, acc[m][j]);
        }
    }
    const int n = n0 + q * 16, left = a.N - n;
    if (left <= 0) continue;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      if (row[j] < 0) continue;
      float v[16] = {};
      if (a.base) load16(a.base, a.base_f32, (size_t)row[j] * a.ldb + n, left, v);
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * m + i] += acc[m][j][i];
      store16<F32>(a.y, (size_t)row[j] * a.ldy + n, left, v);
    }
  }
}

// Chunks that T rows over E groups may make.
int max_chunks(int T, int E) { return (T < E ? T : E) + T / kChunkRows; }

// Slices of K: enough that the first launch has some 512 workgroups, each wave at
// least one block of 128 columns.
constexpr int kInWorkgroups = 512;
int slices_of(int K, int R, int E, int T) {
  const int most = ((K + 127) / 128 + 3) / 4;
  const int s = kInWorkgroups / (max_chunks(T, E) * ((R + kRankTile - 1) / kRankTile));
  return s < 1 ? 1 : s < most ? s : most;
}

}  // namespace

size_t adapters_workspace(int K, int R, int E, int T) {
  // (a call of fewer rows may take more slices: T * slices stays below
  // kInWorkgroups * kChunkRows where there are any)
  const size_t most = ((size_t)((K + 127) / 128) + 3) / 4;
  size_t rows = (size_t)T * most;
  if (rows > (size_t)kInWorkgroups * kChunkRows) rows = (size_t)kInWorkgroups * kChunkRows;
  if (rows < (size_t)T) rows = T;
  return rows * R * 4;
}

hipError_t adapters_forward(const Adapters &a, void *workspace, hipStream_t st) {
  float *u = static_cast<float *>(workspace);
  const int slices = slices_of(a.K, a.R, a.E, a.T);
  const int bare = !(a.base == a.y);
  const dim3 in(max_chunks(a.T, a.E), slices, (a.R + kRankTile - 1) / kRankTile);
  if (a.x_f32)
    hipLaunchKernelGGL(adapters_in_kernel<true>, in, dim3(256), 0, st, a, u, slices);
  else
    hipLaunchKernelGGL(adapters_in_kernel<false>, in, dim3(256), 0, st, a, u, slices);
  const int cols = 4 * kColBlock;
  const dim3 out(max_chunks(a.T, a.E + bare), (a.N + cols - 1) / cols);
  const size_t lds = (size_t)((a.R + 31) / 32) * (a.y_f32 ? 3 : 2) * kTiles * 64 * 16;
  if (a.y_f32)
    hipLaunchKernelGGL(adapters_out_kernel<true>, out, dim3(256), lds, st, a, u, slices, cols,
                       bare);
  else
    hipLaunchKernelGGL(adapters_out_kernel<false>, out, dim3(256), lds, st, a, u, slices, cols,
                       bare);
  return hipGetLastError();
}

}  // namespace cai4
