// rows.hpp -- device helpers: runs of bf16 or f32 values of rows at any alignment.
#pragma once
#include "int4_common.hpp"

namespace cai4 {
namespace {

// V neighbouring values as they are stored: loads or stores of 8 or 16 bytes (32:
// two) aligned as T only.  Rows of odd widths start between words, which
// vector loads and stores allow.
template <class T, int V>
struct Run {
  T v[V];
};
typedef uint32_t u32x4_by1_t __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x4_by2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_by4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_by2_t __attribute__((ext_vector_type(2), aligned(2)));
template <int bytes, int align>
struct Whole;
template <>
struct Whole<16, 1> {
  typedef u32x4_by1_t type;
};
template <>
struct Whole<16, 2> {
  typedef u32x4_by2_t type;
};
template <>
struct Whole<16, 4> {
  typedef u32x4_by4_t type;
};
template <>
struct Whole<8, 2> {
  typedef u32x2_by2_t type;
};
// STREAM: past the caches' replacement, for data that would fill them many times over.
template <class T, int V, bool STREAM = false>
CAI4_DEV Run<T, V> load_run(const T *p) {
  if constexpr (sizeof(T) * V == 32) {
    const Run<T, V / 2> h[2] = {load_run<T, V / 2>(p), load_run<T, V / 2>(p + V / 2)};
    return __builtin_bit_cast(Run<T, V>, h);
  } else {
    typedef typename Whole<sizeof(T) * V, sizeof(T)>::type W;
    const W *w = reinterpret_cast<const W *>(p);
    return __builtin_bit_cast(Run<T, V>, STREAM ? __builtin_nontemporal_load(w) : *w);
  }
}
template <bool STREAM = false, class T, int V>
CAI4_DEV void store_run(T *p, const Run<T, V> &r) {
  typedef typename Whole<sizeof(T) * V, sizeof(T)>::type W;
  W *w = reinterpret_cast<W *>(p);
  if constexpr (STREAM)
    __builtin_nontemporal_store(__builtin_bit_cast(W, r), w);
  else
    *w = __builtin_bit_cast(W, r);
}
// The first n (< V) of them.
template <class T, int V>
CAI4_DEV Run<T, V> load_part(const T *p, int n) {
  Run<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = i < n ? p[i] : T(0);
  return r;
}
template <class T, int V>
CAI4_DEV void store_part(T *p, const Run<T, V> &r, int n) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = r.v[i];
}
// A whole run, or its first n values.  FULL is a constant of the code around: a run
// that may be either is loaded value by value by the compiler.
template <bool FULL, class T, int V, bool STREAM = false>
CAI4_DEV Run<T, V> load_some(const T *p, int n) {
  if constexpr (FULL)
    return load_run<T, V, STREAM>(p);
  else
    return load_part<T, V>(p, n);
}
template <bool FULL, bool STREAM = false, class T, int V>
CAI4_DEV void store_some(T *p, const Run<T, V> &r, int n) {
  if constexpr (FULL)
    store_run<STREAM>(p, r);
  else
    store_part<T, V>(p, r, n);
}

CAI4_DEV float value_of_row(float v) { return v; }
CAI4_DEV float value_of_row(uint16_t v) { return bf16_to_f32(v); }
template <class T>
CAI4_DEV T row_value(float v) {
  if constexpr (sizeof(T) == 2)  // (to nearest even, NaN kept quiet)
    return __builtin_bit_cast(uint16_t, (__bf16)v);
  else
    return v;
}

}  // namespace
}  // namespace cai4
