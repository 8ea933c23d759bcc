// adapters.hip -- low-rank adapters of many requests at once:
//   y_t = base_t + s_a B_a (A_a x_t),  a: row t's adapter (rows without one: base_t)
//
// Rows come sorted by adapter, in chunks of one adapter: 16 to 64 rows in the first
// launch, 32 in the second.  The first is u = A x for every chunk (K in slices where
// chunks are few; their partial sums stay f32), the other y = base + B (s u), which adds
// the slices in order; a chunk without an adapter, or of rank 0, is copied from base.
// (Both in one launch, u made again by every workgroup: one row of rank 16 took 10 us of
// kernel time for 4.9 + 5.4, but rank 32, or 16 rows and more, 15 to 65 % more than two.)
//
// Both products run on bf16 MFMAs with f32 sums.  A and B are bf16; f32 x, and u,
// enter as a sum of three bf16 planes, each what the ones before left over: all 24 bits,
// also where y is bf16, since an f32 base may take away the sum's upper ones.
//
// Bound: HBM, by base and y (x, A and B besides); rows that are few, by two launches of
// some three dependent round trips each.  4,096 rows, rank 32, 4,096 -> 14,336, all
// bf16: u 17.5 us (27 MB of x, and A from the L2), y 57 (235 MB, 4.1 TB/s; the runtime's
// copy of as many bytes takes 44, the rows copied by this kernel for want of adapters
// 48), 67 to 75 in all.  Rank 64: 23 + 81: the second launch's u and B from the L2 cost it
// what the matrix cores do not.  Rank 128: 36 + 172, rank 256: 59 + 300: past 64, B is read
// once per tile of 16 rows, where it is multiplied.  One row, rank 16, 4,096 -> 4,096: 4.9 +
// 5.4.  64 rows of 33 adapters of rank 4 to 64 in f32, 4,096 -> 14,336: 9.7 + 15.1; the
// second reads rows of B of 128 bytes of which the rank fills half.
#include <array>
#include <type_traits>

#include "adapters_common.hpp"
#include "rows.hpp"
#include "tokens.hpp"

namespace cai4 {
namespace {

constexpr int kPlanes = 3;  // of an f32 value

// Eight values as the operands of three MFMAs: bf16 planes, the first one truncated (so
// that no finite value becomes infinite).  It leaves 16 bits, the second half a step of
// its 8, the third the rest: all 24 bits.  An infinity is in the first alone, a NaN in any.
CAI4_DEV void operands_of(const float (&v)[8], u32x4_t (&op)[kPlanes]) {
  auto pair = [](float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i], b = v[2 * i + 1];
    op[0][i] = __builtin_amdgcn_perm(fbits(b), fbits(a), 0x07060302u);
    float ra = a - bitsf(fbits(a) & 0xFFFF0000u), rb = b - bitsf(fbits(b) & 0xFFFF0000u);
    ra = fabsf(a) == INFINITY ? 0.f : ra;
    rb = fabsf(b) == INFINITY ? 0.f : rb;
    op[1][i] = pair(ra, rb);
    op[2][i] = pair(ra - bitsf(op[1][i] << 16), rb - bitsf(op[1][i] & 0xFFFF0000u));
  }
}

// What an infinity w meets in planes: 0 times it in those that a value leaves empty, or
// two infinities of unlike sign, both NaN.  So where a sum comes out as NaN it is taken
// again, with the infinities (and NaN) of each side apart, times the other side's signs;
// the other sums of the wave keep their bits, to which it adds zeros.  Each function
// takes words of two bf16 values.
CAI4_DEV uint32_t halves_of(uint32_t tops) { return ((tops & 0x80008000u) >> 15) * 0xFFFFu; }
CAI4_DEV uint32_t nonfinite(uint32_t w) { return halves_of((w & 0x7F807F80u) + 0x00800080u); }
CAI4_DEV uint32_t nonzero(uint32_t w) { return halves_of((w & 0x7FFF7FFFu) + 0x7FFF7FFFu); }
CAI4_DEV uint32_t sign_of(uint32_t w) { return nonzero(w) & ((w & 0x80008000u) | 0x3F803F80u); }
struct Sides {
  u32x4_t finite, infinite, sign;
};
CAI4_DEV Sides sides_of(u32x4_t w) {
  Sides s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s.infinite[i] = w[i] & nonfinite(w[i]);
    s.finite[i] = w[i] & ~nonfinite(w[i]);
    s.sign[i] = sign_of(w[i]);
  }
  return s;
}
// The same of a value's planes, the first of which alone says whether it is finite; an
// infinite one leaves them.
CAI4_DEV Sides sides_of(u32x4_t (&op)[kPlanes]) {
  Sides s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t infinite = nonfinite(op[0][i]);
    uint32_t first = op[kPlanes - 1][i];  // of the planes, the first that is not zero
#pragma unroll
    for (int p = kPlanes - 2; p >= 0; --p)
      first = (op[p][i] & nonzero(op[p][i])) | (first & ~nonzero(op[p][i]));
    s.infinite[i] = op[0][i] & infinite;
    s.sign[i] = sign_of(first);
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) op[p][i] &= ~infinite;
  }
  return s;
}
// acc + w times a value in planes, of sides s.  (One at a time: few registers, since the
// kernels that may come here need theirs for loads in flight.)
CAI4_DEV void add_sides(u32x4_t w, const u32x4_t (&op)[kPlanes], const Sides &s, f32x4_t &acc) {
  const Sides ws = sides_of(w);
#pragma unroll
  for (int p = 0; p < kPlanes; ++p) acc = mfma_bf16(ws.finite, op[p], acc);
  acc = mfma_bf16(ws.infinite, s.sign, acc);
  acc = mfma_bf16(ws.sign, s.infinite, acc);
  __builtin_amdgcn_sched_barrier(0);
}
// Whether any lane has a NaN.
template <int N>
CAI4_DEV bool any_nan(const f32x4_t (&acc)[N]) {
  bool nan = false;
#pragma unroll
  for (int i = 0; i < N; ++i)
    nan |= __builtin_isunordered(acc[i][0], acc[i][1]) || __builtin_isunordered(acc[i][2], acc[i][3]);
  return __builtin_expect(__ballot(nan) != 0, 0);
}

// Bits to keep of columns r .. r + 7 of a row of B: those below the rank (the others
// may hold anything).
CAI4_DEV u32x4_t keep_of(int rank, int r) {
  u32x4_t m;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m[i] = (r + 2 * i < rank ? 0xFFFFu : 0u) | (r + 2 * i + 1 < rank ? 0xFFFF0000u : 0u);
  return m;
}

// ---- u = A x ----

constexpr int kInWaves = 8;  // of a workgroup: each has its own columns

// A wave's sums over blocks [b0, b1) of 128 columns with infinities apart (f32 x).
template <int RT, int NT>
CAI4_DEV void sums_of_sides(const Adapters &a, const uint16_t *const (&A)[RT],
                            const uint8_t *const (&x)[NT], int b0, int b1,
                            f32x4_t (&acc)[RT][NT]) {
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int q = (threadIdx.x & 63) >> 4;
  for (int at = b0 * 128; at < b1 * 128; at += 32) {
    const bool in = at + q * 8 < a.K;
    const int col = in ? at + q * 8 : 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const Run<float, 8> r = load_run<float, 8>(reinterpret_cast<const float *>(x[j]) + col);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)  // (quiet: the first plane of a NaN is one)
        v[i] = in ? __builtin_canonicalizef(r.v[i]) : 0.f;
      u32x4_t op[kPlanes];
      operands_of(v, op);
      const Sides s = sides_of(op);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        u32x4_t w = *reinterpret_cast<const u32x4_t *>(A[i] + col);
        w = in ? w : u32x4_t{0, 0, 0, 0};
        add_sides(w, op, s, acc[i][j]);
      }
    }
  }
}

// A workgroup's slice of K for RT * 16 ranks and NT * 16 rows of a chunk.  A wave has
// blocks [b0, b1) of 128 columns; the waves' sums are added in LDS, eight to four to
// one.  Rows and ranks past the last ones repeat a valid one: nobody reads their sums.
template <bool F32, int RT, int NT>
CAI4_DEV void adapters_in_chunk(const Adapters &a, const Chunk &ch, int rank, int r0, int b0, int b1,
                                f32x4_t (*part)[RT * NT][64], float *u) {
  constexpr int P = F32 ? kPlanes : 1;
  constexpr int S = F32 && NT > 1 ? 2 : 4;  // steps of 32 columns loaded at a time
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
  const uint16_t *A[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = r0 + i * 16 + c;
    A[i] = a.a + ((size_t)ch.group * a.R + (r < rank ? r : r0)) * a.K;
  }
  const uint8_t *x[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int k = i * 16 + c;
    const int t = row_of(a, ch, k < ch.rows ? k : 0);
    x[i] = static_cast<const uint8_t *>(a.x) + (size_t)(t < 0 ? 0 : t) * a.ldx;
  }
  f32x4_t acc[RT][NT] = {};
  for (int at = b0 * 128; at < b1 * 128; at += S * 32) {
    const bool whole = at + S * 32 <= a.K;
    u32x4_t av[S][RT], xv[S][NT];
    f32x4_t xf[S][NT][2];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      int col = at + s * 32 + q * 8;
      col = whole || col < a.K ? col : 0;
#pragma unroll
      for (int i = 0; i < RT; ++i) av[s][i] = *reinterpret_cast<const u32x4_t *>(A[i] + col);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if constexpr (F32) {
          const float *p = reinterpret_cast<const float *>(x[i]) + col;
          xf[s][i][0] = __builtin_bit_cast(f32x4_t, load_run<float, 4>(p));
          xf[s][i][1] = __builtin_bit_cast(f32x4_t, load_run<float, 4>(p + 4));
        } else {
          xv[s][i] = __builtin_bit_cast(
              u32x4_t, load_run<uint16_t, 8>(reinterpret_cast<const uint16_t *>(x[i]) + col));
        }
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (!whole) {  // columns past the last: zero on both sides
        const bool in = at + s * 32 + q * 8 < a.K;
#pragma unroll
        for (int i = 0; i < RT; ++i) av[s][i] = in ? av[s][i] : u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if constexpr (F32) {
            xf[s][i][0] = in ? xf[s][i][0] : f32x4_t{0.f, 0.f, 0.f, 0.f};
            xf[s][i][1] = in ? xf[s][i][1] : f32x4_t{0.f, 0.f, 0.f, 0.f};
          } else {
            xv[s][i] = in ? xv[s][i] : u32x4_t{0, 0, 0, 0};
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        u32x4_t op[P];
        if constexpr (F32) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = xf[s][j][i / 4][i % 4];
          operands_of(v, op);
        } else {
          op[0] = xv[s][j];
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int p = 0; p < P; ++p) acc[i][j] = mfma_bf16(av[s][i], op[p], acc[i][j]);
      }
    }
  }
  if constexpr (F32) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < RT; ++i) nan |= any_nan(acc[i]);
    if (nan) sums_of_sides(a, A, x, b0, b1, acc);
  }
  constexpr int kHalf = kInWaves / 2;
  if (wave >= kHalf)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) part[wave - kHalf][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  if (wave < kHalf)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] += acc[i][j];
  __syncthreads();
  // tile i, j: lane holds ranks r0 + 16 i + 4 q + [0, 4) of row 16 j + c
  for (int k = wave; k < RT * NT; k += kInWaves) {
    f32x4_t v = part[0][k][lane];
#pragma unroll
    for (int w = 1; w < kHalf; ++w) v += part[w][k][lane];
    const int r = r0 + k / NT * 16 + q * 4, row = k % NT * 16 + c;
    if (r < a.R && row < ch.rows)
      *reinterpret_cast<f32x4_t *>(u + (size_t)(ch.row0 + row) * a.R + r) = v;
  }
}

template <bool F32, int RT, int NT>
__global__ __launch_bounds__(64 * kInWaves) void adapters_in_kernel(Adapters a, float *u,
                                                                    int slices) {
  __shared__ f32x4_t part[kInWaves / 2][RT * NT][64];
  const int wave = threadIdx.x >> 6;
  const Chunk ch = find_chunk<16 * NT>(a, blockIdx.x, false);
  if (ch.rows == 0) return;
  const int rank = rank_of(a, ch.group), r0 = blockIdx.z * RT * 16;
  if (r0 >= rank) return;
  const int slice = blockIdx.y;
  const int blocks = (a.K + 127) / 128, parts = slices * kInWaves, me = slice * kInWaves + wave;
  const int b0 = (int)((int64_t)blocks * me / parts), b1 = (int)((int64_t)blocks * (me + 1) / parts);
  adapters_in_chunk<F32, RT, NT>(a, ch, rank, r0, b0, b1, part, u + (size_t)slice * a.T * a.R);
}

// ---- y = base + B (s u) ----

constexpr int kOutWaves = 4, kColBlock = 64;  // columns of a wave at a time
// Rows of a chunk.  32 / 64 / 128: 256 rows of as many adapters 24.2 / 25.6 / 30.1 us, 8,192 of
// rank 32 60.7 / 65.4 / 70.5, 4,096 of rank 64 100 / 102 / 114.
constexpr int kOutRows = 32;

enum BaseType { kBaseNone, kBaseBf16, kBaseF32 };

// Outputs leave the MFMAs as 16 columns of row c in lane (c, q), in RUNS runs of 16
// bytes (of y's type).  Four lanes' runs of one row are 64 bytes, half a line; lanes c
// and c ^ 1 exchange every second run, so that a store writes whole lines of the
// eight even rows, the next those of the odd ones (4,096 x 14,336 in bf16, copied so past
// the caches: 48 us, in half lines 56).  f32: run m is columns 16 m + 4 q of the block,
// tile m; bf16: run h is 32 h + 8 q, tiles 2 h and 2 h + 1 with four columns each in
// turn.
template <bool F32>
CAI4_DEV int weight_col(int m, int c) {
  return F32 ? m * 16 + c : (m >> 1) * 32 + (c >> 2) * 8 + (m & 1) * 4 + (c & 3);
}
// Lane c ^ 1's value.
CAI4_DEV float of_pair(float v) { return dpp_f32<0xB1>(v); }

// What a block of 64 columns of NT * 16 rows reads: base, and B's rows (STEPS of 32
// ranks; 0: as many as there are, read where they are multiplied).  Run i of tile j of
// a lane is of row pair_row[j][i & 1] (-1: none), columns run_col(i) on.
template <bool F32, int BASE, int STEPS, int NT>
struct OutBlock {
  static constexpr int P = kPlanes, V = F32 ? 4 : 8, RUNS = 16 / V;
  typedef typename std::conditional<F32, float, uint16_t>::type Y;
  typedef typename std::conditional<BASE == kBaseF32, float, uint16_t>::type X;
  Run<X, V> base[NT][RUNS];
  u32x4_t bv[STEPS ? STEPS : 1][4];

  // Runs 2 i and 2 i + 1 of a lane after the exchange: both of the even lane's run 2 i
  // (c even) or run 2 i + 1 (c odd), of the even row and of the odd one.
  static CAI4_DEV int run_col(int i) {
    const int lane = threadIdx.x & 63;
    return ((i & ~1) + (lane & 1)) * (kColBlock / RUNS) + (lane >> 4) * V;
  }

  // Ranks step * 32 + 8 q on of row m's column of B.
  template <bool FULL>
  static CAI4_DEV const u32x4_t *weights_at(const Adapters &a, const uint16_t *B, int n0, int step,
                                            int m) {
    const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4, left = a.N - n0;
    const int r = step * 32 + q * 8, at = weight_col<F32>(m, c);
    const int n = FULL || at < left ? n0 + at : a.N - 1;
    return reinterpret_cast<const u32x4_t *>(B + (size_t)n * a.R + (r < a.R ? r : 0));
  }
  template <bool FULL>
  CAI4_DEV void load_b(const Adapters &a, const uint16_t *B, int n0, int step, u32x4_t (&v)[4]) {
#pragma unroll
    for (int m = 0; m < 4; ++m) v[m] = *weights_at<FULL>(a, B, n0, step, m);
  }
  // Row r of p, made anew at each use: eight addresses kept would be 16 registers.
  template <class T>
  static CAI4_DEV T *row_at(T *p, uint32_t ld, int r) {
    uint32_t t = r < 0 ? 0 : r;
    asm volatile("" : "+v"(t));
    typedef typename std::conditional<std::is_const<T>::value, const uint8_t, uint8_t>::type B;
    return reinterpret_cast<T *>(reinterpret_cast<B *>(p) + (uint64_t)t * ld);
  }
  template <bool FULL>
  CAI4_DEV void load(const Adapters &a, const uint16_t *B, const int (&row)[NT][2], int n0) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) load_b<FULL>(a, B, n0, s, bv[s]);
    load_base<FULL>(a, row, n0);
  }
  template <bool FULL>
  CAI4_DEV void load_base(const Adapters &a, const int (&row)[NT][2], int n0) {
    const int left = a.N - n0;
    if constexpr (BASE != kBaseNone) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const X *p = row_at(static_cast<const X *>(a.base) + n0, a.ldb, row[j][h]);
#pragma unroll
          for (int i = h; i < RUNS; i += 2) {
            const int at = run_col(i);
            if constexpr (FULL)
              base[j][i] = load_run<X, V>(p + at);
            else
              base[j][i] = load_part<X, V>(p + at, left - at);
          }
        }
    }
  }
  template <bool FULL, bool STREAM>
  static CAI4_DEV void store(const Adapters &a, int row, int n0, int at, const Run<Y, V> &y) {
    if (row < 0) return;
    Y *p = row_at(static_cast<Y *>(a.y) + n0, a.ldy, row) + at;
    if constexpr (FULL)
      store_run<STREAM>(p, y);
    else
      store_part<Y, V>(p, y, a.N - n0 - at);
  }
  // y = base, every bit of it where both are of one type.
  template <bool FULL, bool STREAM>
  CAI4_DEV void copy(const Adapters &a, const int (&row)[NT][2], int n0) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        Run<Y, V> y = {};
#pragma unroll
        for (int k = 0; k < V; ++k) {
          if constexpr (BASE == kBaseNone)
            continue;
          else if constexpr (std::is_same<X, Y>::value)
            y.v[k] = base[j][i].v[k];
          else
            y.v[k] = row_value<Y>(value_of_row(base[j][i].v[k]));
        }
        store<FULL, STREAM>(a, row[j][i & 1], n0, run_col(i), y);
      }
  }
  CAI4_DEV void keep_ranks(int rank) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const u32x4_t keep = keep_of(rank, s * 32 + (threadIdx.x & 63) / 16 * 8);
#pragma unroll
      for (int m = 0; m < 4; ++m) bv[s][m] &= keep;
    }
  }
  // The sums of tile j's rows with infinities apart.
  template <bool FULL>
  static CAI4_DEV void sums_of_sides(const Adapters &a, const uint16_t *B, int steps, int rank,
                                     const u32x4_t *us, int j, int n0, f32x4_t (&acc)[4]) {
    const int lane = threadIdx.x & 63, q = lane >> 4;
#pragma unroll
    for (int m = 0; m < 4; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      u32x4_t op[P];
#pragma unroll
      for (int p = 0; p < P; ++p) op[p] = us[((s * P + p) * NT + j) * 64 + lane];
      const Sides sides = sides_of(op);
      const u32x4_t keep = keep_of(rank, s * 32 + q * 8);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const u32x4_t w = *weights_at<FULL>(a, B, n0, s, m);
        add_sides(w & keep, op, sides, acc[m]);
      }
    }
  }
  // (A tile of 16 rows at a time: fewer sums at once, more waves.)
  template <bool FULL, bool STREAM>
  CAI4_DEV void finish(const Adapters &a, const uint16_t *B, int steps, int rank, const u32x4_t *us,
                       const int (&row)[NT][2], int n0) {
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const bool odd = lane & 1;
    keep_ranks(rank);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      f32x4_t acc[4] = {};
      auto add = [&](int step, const u32x4_t (&v)[4]) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const u32x4_t uv = us[((step * P + p) * NT + j) * 64 + lane];
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[m] = mfma_bf16(v[m], uv, acc[m]);
        }
      };
      if constexpr (STEPS > 0) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) add(s, bv[s]);
      } else {
        for (int s = 0; s < steps; ++s) {
          const u32x4_t keep = keep_of(rank, s * 32 + q * 8);
          load_b<FULL>(a, B, n0, s, bv[0]);
#pragma unroll
          for (int m = 0; m < 4; ++m) bv[0][m] &= keep;
          add(s, bv[0]);
        }
      }
      if (any_nan(acc)) {
        // (what was loaded is loaded again: it and its addresses, kept meanwhile, would
        // take registers)
        int again = n0;
        asm volatile("" : "+v"(again));
        sums_of_sides<FULL>(a, B, steps, rank, us, j, again, acc);
        load<FULL>(a, B, row, again);
        keep_ranks(rank);
      }
#pragma unroll
      for (int i = 0; i < RUNS; i += 2) {
        __builtin_amdgcn_sched_barrier(0);  // (one pair of runs at a time: registers)
        Run<Y, V> y[2];  // of the even row, of the odd one
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float lo = acc[i * (V / 4) + k / 4][k % 4];
          const float hi = acc[(i + 1) * (V / 4) + k / 4][k % 4];
          const float got = of_pair(odd ? lo : hi);
          const float d[2] = {odd ? got : lo, odd ? hi : got};
#pragma unroll
          for (int h = 0; h < 2; ++h)
            y[h].v[k] = row_value<Y>(
                BASE == kBaseNone ? d[h] : value_of_row(base[j][i + h].v[k]) + d[h]);
        }
        const int at = run_col(i);
#pragma unroll
        for (int h = 0; h < 2; ++h) store<FULL, STREAM>(a, row[j][h], n0, at, y[h]);
      }
    }
  }
};

// A chunk's NT * 16 rows over columns [n_begin, n_end), a block of 64 per wave at a
// time.  The first loads are issued before u is read.
template <bool F32, int BASE, int STEPS, int NT, bool STREAM>
CAI4_DEV void adapters_out_chunk(const Adapters &a, const Chunk &ch, const float *u, int slices,
                                 int n_begin, int n_end, u32x4_t *us) {
  constexpr int P = kPlanes, kStride = kOutWaves * kColBlock;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, q = lane >> 4;
  const bool own = ch.group < a.E;
  const int rank = own ? rank_of(a, ch.group) : 0, steps = STEPS ? STEPS : (rank + 31) / 32;
  const float scale = own && a.scales ? a.scales[ch.group] : 1.0f;
  int row[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) row[j][h] = row_of(a, ch, j * 16 + (c & ~1) + h);
  const uint16_t *B = a.b + (size_t)(own ? ch.group : 0) * a.N * a.R;
  int n0 = n_begin + wave * kColBlock;
  const int n_full = n_end < a.N ? n_end : a.N / kColBlock * kColBlock;  // end of whole blocks
  OutBlock<F32, BASE, STEPS, NT> now;
  if (rank == 0) {  // no product: base + 0 would lose the sign of a zero
    if (a.base == a.y) return;
    for (; n0 < n_full; n0 += kStride) {
      now.template load_base<true>(a, row, n0);
      now.template copy<true, STREAM>(a, row, n0);
    }
    if (n0 < n_end && n0 < a.N) {
      now.template load_base<false>(a, row, n0);
      now.template copy<false, false>(a, row, n0);
    }
    return;
  }
  if (n0 < n_full) now.template load<true>(a, B, row, n0);
  for (int k = wave; k < steps * NT; k += kOutWaves) {
    const int step = k / NT, j = k % NT;
    const int r = step * 32 + q * 8, i0 = j * 16 + c;
    float v[8] = {};
    if (i0 < ch.rows && r < rank) {
      const float *p = u + (size_t)(ch.row0 + i0) * a.R + r;
      const size_t stride = (size_t)a.T * a.R;
      for (int h0 = 0; h0 < slices; h0 += 4) {  // (in order; four slices' loads at a time)
        f32x4_t t[4][2];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float *s = p + (h0 + h < slices ? h0 + h : h0) * stride;
          t[h][0] = reinterpret_cast<const f32x4_t *>(s)[0];
          t[h][1] = reinterpret_cast<const f32x4_t *>(s)[1];
        }
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += h0 + h < slices ? t[h][i / 4][i % 4] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r + i < rank ? v[i] * scale : 0.f;
    }
    u32x4_t op[P];
    operands_of(v, op);
#pragma unroll
    for (int p = 0; p < P; ++p) us[((step * P + p) * NT + j) * 64 + lane] = op[p];
  }
  __syncthreads();
  while (n0 < n_full) {
    now.template finish<true, STREAM>(a, B, steps, rank, us, row, n0);
    n0 += kStride;
    if (n0 < n_full) now.template load<true>(a, B, row, n0);
  }
  if (n0 < n_end && n0 < a.N) {  // the last columns
    now.template load<false>(a, B, row, n0);
    now.template finish<false, false>(a, B, steps, rank, us, row, n0);
  }
}

// (Ranks past 64, whose B is read where it is multiplied, want four waves per SIMD rather
// than three: 2,048 rows of rank 96, 4,096 -> 4,096, 33 / 36 us.  Fewer ranks do not fit
// four, for lack of registers.)
template <bool F32, int BASE, int STEPS>
__global__ __launch_bounds__(64 * kOutWaves, STEPS ? 1 : 4) void adapters_out_kernel(
    Adapters a, const float *u, int slices, int cols, int bare, int stream) {
  extern __shared__ u32x4_t us[];  // [steps of 32 ranks][planes][tiles][lane]
  const Chunk ch = find_chunk<kOutRows>(a, blockIdx.y, bare);
  if (ch.rows == 0) return;
  const int n0 = blockIdx.x * cols, n1 = n0 + cols < a.N ? n0 + cols : a.N;
  if (ch.rows <= 16)
    adapters_out_chunk<F32, BASE, STEPS, 1, false>(a, ch, u, slices, n0, n1, us);
  else if (stream)
    adapters_out_chunk<F32, BASE, STEPS, kOutRows / 16, true>(a, ch, u, slices, n0, n1, us);
  else
    adapters_out_chunk<F32, BASE, STEPS, kOutRows / 16, false>(a, ch, u, slices, n0, n1, us);
}

// Chunks of `rows` rows that T rows over E groups may make.
int max_chunks(int T, int E, int rows) { return (T < E ? T : E) + T / rows; }

// Rows of a chunk of the first launch: more of them read A less often, fewer make more
// workgroups.  16 / 32 / 64 rows, nine adapters, us of the whole call: 512 rows of rank 32
// 20.9 / 22.6 / 24.6; 1,024 of rank 16 19.2 / 18.2 / 20.5; 4,096 of rank 32 80 / 75 / 77;
// 2,048 of rank 64 40.4 / 40.4 / 35.0, 4,096 of it 111 / 107 / 102.  (By T and R alone: with
// 256 adapters a chunk of 32 holds some eight of 2,048 rows; rank 32, 4,096 -> 4,096, 17 us
// of the call's 36.)
// Slices of K, each read again by the second launch: up to some 1,024 workgroups, each
// wave at least one block of 128 columns.  1,024 / 512 / 256: 256 adapters' rows 23.9 / 27.3 /
// 27.4, 8,192 rows of rank 32 60.8 / 66.1 / 66.2, 4,096 of rank 64 99.9 / 99.6 / 96.2.
constexpr int kInWorkgroups = 1024;
int in_tiles(int R, int T) { return T < 1024 ? 1 : R > 32 && T >= 2048 ? 4 : 2; }
int rank_tiles(int R) { return R <= 16 ? 1 : R <= 32 ? 2 : 4; }  // of a workgroup
int rank_groups(int R) { return (R + 16 * rank_tiles(R) - 1) / (16 * rank_tiles(R)); }
int slices_of(int K, int R, int E, int T) {
  const int most = ((K + 127) / 128 + kInWaves - 1) / kInWaves;
  const int s = kInWorkgroups / (max_chunks(T, E, 16 * in_tiles(R, T)) * rank_groups(R));
  return s < 1 ? 1 : s < most ? s : most;
}

// Outputs of 64 MiB and more, in whole lines, are written past the caches, so or not:
// 117 MB 74.9 / 78.7 us, 67 MB 55.2 / 61.7.  (15 MB: 19.4 / 21.3, but what reads those next
// finds them there.)
constexpr size_t kStreamBytes = (size_t)64 << 20, kLine = 128;

// Columns of a workgroup of the second launch: whole rounds of its waves, for some 3,072
// workgroups.  1,536 / 3,072 / 6,144: 4,096 rows of rank 32 81 / 75 / 74 us, 64 rows of mixed
// ranks 27.3 / 27.0 / 32.9.
constexpr int kOutWorkgroups = 3072;
int cols_of(int N, int chunks) {
  const int each = kOutWaves * kColBlock, blocks = (N + each - 1) / each;
  const int per = (int)(((int64_t)blocks * chunks + kOutWorkgroups - 1) / kOutWorkgroups);
  return each * (per < 1 ? 1 : per < blocks ? per : blocks);
}

template <bool F32, int BASE, int STEPS>
void launch_out(const Adapters &a, const float *u, int slices, int bare, hipStream_t st) {
  const int chunks = max_chunks(a.T, a.E + bare, kOutRows), cols = cols_of(a.N, chunks);
  const int stream = (size_t)a.T * a.N * (F32 ? 4 : 2) >= kStreamBytes && a.ldy % kLine == 0 &&
                     (uintptr_t)a.y % kLine == 0;
  const size_t lds = (size_t)((a.R + 31) / 32) * kPlanes * (kOutRows / 16) * 64 * 16;
  hipLaunchKernelGGL((adapters_out_kernel<F32, BASE, STEPS>),
                     dim3((a.N + cols - 1) / cols, chunks), dim3(64 * kOutWaves), lds, st, a, u,
                     slices, cols, bare, stream);
}
template <bool F32, int BASE>
void launch_out(const Adapters &a, const float *u, int slices, int bare, hipStream_t st) {
  if (a.R <= 32)
    launch_out<F32, BASE, 1>(a, u, slices, bare, st);
  else if (a.R <= 64)
    launch_out<F32, BASE, 2>(a, u, slices, bare, st);
  else
    launch_out<F32, BASE, 0>(a, u, slices, bare, st);
}
template <bool F32>
void launch_out(const Adapters &a, const float *u, int slices, int bare, hipStream_t st) {
  if (!a.base)
    launch_out<F32, kBaseNone>(a, u, slices, bare, st);
  else if (a.base_f32)
    launch_out<F32, kBaseF32>(a, u, slices, bare, st);
  else
    launch_out<F32, kBaseBf16>(a, u, slices, bare, st);
}

template <bool F32, int RT>
void launch_in(const Adapters &a, float *u, int slices, hipStream_t st) {
  const int tiles = in_tiles(a.R, a.T);
  const dim3 grid(max_chunks(a.T, a.E, 16 * tiles), slices, rank_groups(a.R)),
      block(64 * kInWaves);
  if (tiles == 1)
    hipLaunchKernelGGL((adapters_in_kernel<F32, RT, 1>), grid, block, 0, st, a, u, slices);
  else if (tiles == 2)
    hipLaunchKernelGGL((adapters_in_kernel<F32, RT, 2>), grid, block, 0, st, a, u, slices);
  else
    hipLaunchKernelGGL((adapters_in_kernel<F32, RT, 4>), grid, block, 0, st, a, u, slices);
}
template <bool F32>
void launch_in(const Adapters &a, float *u, int slices, hipStream_t st) {
  const int rt = rank_tiles(a.R);
  if (rt == 1)
    launch_in<F32, 1>(a, u, slices, st);
  else if (rt == 2)
    launch_in<F32, 2>(a, u, slices, st);
  else
    launch_in<F32, 4>(a, u, slices, st);
}

}  // namespace

size_t adapters_workspace(int K, int R, int E, int T) {
  // (a call of fewer rows may take more slices: T * slices stays below
  // kInWorkgroups * 64 where there are several)
  const size_t most = ((size_t)((K + 127) / 128) + kInWaves - 1) / kInWaves;
  size_t rows = (size_t)T * most;
  if (rows > (size_t)kInWorkgroups * 64) rows = (size_t)kInWorkgroups * 64;
  if (rows < (size_t)T) rows = T;
  return rows * R * 4;
}

hipError_t adapters_forward(const Adapters &a, void *workspace, hipStream_t st) {
  float *u = static_cast<float *>(workspace);
  const int slices = slices_of(a.K, a.R, a.E, a.T);
  if (a.x_f32)
    launch_in<true>(a, u, slices, st);
  else
    launch_in<false>(a, u, slices, st);
  const int bare = a.base != a.y;  // (in place: rows without an adapter stay)
  if (a.y_f32)
    launch_out<true>(a, u, slices, bare, st);
  else
    launch_out<false>(a, u, slices, bare, st);
  return hipGetLastError();
}

}  // namespace cai4
