// Tokens sorted by expert and back, and low-rank adapters, through the C++ host API
// (include/cascadia_int4.hpp), with small whole numbers whose results are exact.
//
// Prints one line per check and "cpp tokens: N checks OK"; exit status 1 on the first
// failure.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>

#include "cascadia_int4.hpp"

namespace ci = cascadia_int4;

namespace {

int g_checks = 0;

void expect(bool ok, const std::string &what) {
  if (!ok) {
    std::printf("FAIL %s\n", what.c_str());
    std::fflush(stdout);
    std::exit(1);
  }
  ++g_checks;
  std::printf("ok   %s\n", what.c_str());
}

template <class T>
ci::DeviceBuffer<T> on_device(const std::vector<T> &v) {
  ci::DeviceBuffer<T> b(v.size());
  b.upload(v.data());
  return b;
}

template <class F>
bool refused(F f) {
  try {
    f();
  } catch (const std::invalid_argument &) {
    return true;
  }
  return false;
}

uint16_t bf16(float v) { return ci::f32_to_bf16_bits(v); }
using CF = ci::DeviceSlice<const float>;
using CH = ci::DeviceSlice<const uint16_t>;

}  // namespace

int main() {
  const size_t t = 3, k = 2, e = 4, cols = 5, n = t * k;
  const auto ids = on_device(std::vector<int32_t>{2, 0, -1, 2, 0, 3});
  const auto w = on_device(std::vector<float>{0.5f, 1.f, 1.f, 2.f, 4.f, 0.f});
  ci::DeviceBuffer<int32_t> off(e + 1), slots(n), rows(n);
  ci::sort_tokens(ids, k, e, off, slots, rows);
  expect(off.download() == std::vector<int32_t>({0, 2, 2, 4, 5}), "sort_tokens: offsets");
  expect(slots.download() == std::vector<int32_t>({1, 4, 0, 3, 5, 2}), "sort_tokens: slots");
  expect(rows.download() == std::vector<int32_t>({2, 0, -1, 3, 1, 4}), "sort_tokens: rows");
  ci::sort_tokens(ids, k, e, off, slots, rows, w, 0.25f);
  expect(off.download() == std::vector<int32_t>({0, 2, 2, 4, 4}) &&
             rows.download() == std::vector<int32_t>({2, 0, -1, 3, 1, -1}),
         "sort_tokens: small weights left out");
  expect(refused([&] { ci::sort_tokens(ids, 4, e, off, slots, rows); }) &&
             refused([&] { ci::sort_tokens(ids, k, e + 1, off, slots, rows); }),
         "sort_tokens: wrong lengths refused");

  std::vector<float> x(t * cols), start(n * cols, -7.f);
  for (size_t i = 0; i < x.size(); ++i) x[i] = (float)i + 1;
  const auto xd = on_device(x);
  const auto xs = on_device(start);
  ci::gather_tokens(CF(xd), rows, k, cols, ci::DeviceSlice<float>(xs.slice()));
  {
    const int from[n] = {0, 2, 0, 1, -1, -1};
    const auto v = xs.download();
    bool ok = true;
    for (size_t r = 0; r < n; ++r)
      for (size_t c = 0; c < cols; ++c)
        ok = ok && v[r * cols + c] == (from[r] < 0 ? -7.f : x[from[r] * cols + c]);
    expect(ok, "gather_tokens: rows in order, the others left");
  }
  ci::DeviceBuffer<uint16_t> half(n * cols);
  ci::gather_tokens(CF(xd), rows, k, cols, half.slice());
  expect(half.download()[2 * cols + 4] == bf16(5.f), "gather_tokens: f32 to bf16");
  const auto codes = on_device(std::vector<uint8_t>(t * cols, 9));
  const auto moved = on_device(std::vector<uint8_t>(n * cols, 1));
  ci::gather_tokens(ci::Fp8Rows(codes, {}), rows, k, cols, ci::DeviceSlice<uint8_t>(moved.slice()));
  expect(moved.download()[0] == 9 && moved.download()[4 * cols] == 1, "gather_tokens: codes");

  const ci::Fp8Rows res{CF(xd)};
  ci::DeviceBuffer<float> out(t * cols);
  ci::combine_tokens(CF(xs), rows, k, cols, out.slice(), w, &res);
  {
    const float each[t] = {1.f + 0.5f + 1.f, 1.f + 2.f, 1.f + 4.f};
    const auto v = out.download();
    bool ok = true;
    for (size_t i = 0; i < v.size(); ++i) ok = ok && v[i] == each[i / cols] * x[i];
    expect(ok, "combine_tokens: weighted sums and the residual");
  }
  ci::gather_tokens_grad(CF(xs), rows, k, cols, out.slice());
  expect(out.download()[0] == 2 * x[0] && out.download()[2 * cols] == x[2 * cols],
         "gather_tokens_grad");
  const auto dys = on_device(start);
  ci::DeviceBuffer<float> dw(n);
  ci::combine_tokens_grad(CF(xd), CF(xs), rows, w, k, cols, ci::DeviceSlice<float>(dys.slice()), dw);
  {
    const auto g = dys.download(), d = dw.download();
    float sq[t] = {};
    for (size_t i = 0; i < x.size(); ++i) sq[i / cols] += x[i] * x[i];
    expect(g[2 * cols] == 0.5f * x[0] && g[3 * cols + 1] == 2.f * x[cols + 1] &&
               g[5 * cols] == -7.f,
           "combine_tokens_grad: rows");
    expect(d[0] == sq[0] && d[2] == 0.f && d[3] == sq[1] && d[5] == 0.f,
           "combine_tokens_grad: weights");
  }
  expect(refused([&] { ci::combine_tokens(CF(xs), rows, k, cols + 1, out.slice()); }) &&
             refused([&] { ci::gather_tokens(CF(xd), rows, k, cols, out.slice()); }),
         "rows: wrong lengths refused");

  {  // adapters: a sums the row, b spreads it; scale 2 for the second one
    const size_t na = 2, r = 8, nr = 20, kc = 16;
    std::vector<uint16_t> a(na * r * kc, bf16(0.f)), b(na * nr * r, bf16(0.f));
    for (size_t i = 0; i < na; ++i) {
      for (size_t c = 0; c < kc; ++c) a[i * r * kc + c] = bf16(1.f);
      for (size_t j = 0; j < nr; ++j) b[(i * nr + j) * r] = bf16((float)(j + i));
    }
    const auto ad = on_device(a), bd = on_device(b);
    const auto sc = on_device(std::vector<float>{1.f, 2.f});
    const auto rk = on_device(std::vector<int32_t>{1, 8});
    const ci::Adapters ad2(CH(ad), CH(bd), na, r, nr, kc, rk, sc);
    const auto rid = on_device(std::vector<int32_t>{1, -1, 0});
    ci::DeviceBuffer<int32_t> ao(na + 1), as(t), ar(t);
    ci::sort_tokens(rid, 1, na, ao, as, ar);
    const auto xr = on_device(std::vector<uint16_t>(t * kc, bf16(0.5f)));  // sums of 8
    const auto base = on_device(std::vector<float>(t * nr, 100.f));
    const ci::Fp8Rows bs{CF(base)};
    ci::DeviceBuffer<float> y(t * nr);
    ci::adapters_forward(ad2, CH(xr), ao, as, y.slice(), &bs);
    const auto v = y.download();
    bool ok = true;
    for (size_t j = 0; j < nr; ++j)
      ok = ok && v[j] == 100.f + 16.f * (float)(j + 1) && v[nr + j] == 100.f &&
           v[2 * nr + j] == 100.f + 8.f * (float)j;
    expect(ok, "adapters_forward: two adapters and a row without one");
    ci::DeviceBuffer<uint16_t> h(t * nr);
    ci::adapters_forward(ad2, CH(xr), ao, as, h.slice());
    expect(h.download()[3] == bf16(64.f) && h.download()[nr] == 0, "adapters_forward: no base");
    expect(refused([&] { ci::adapters_forward(ad2, CH(xr), ao, as, out.slice()); }) &&
               refused([&] { ci::Adapters bad(CH(ad), CH(bd), na, 12, nr, kc); }),
           "adapters: wrong lengths and ranks refused");
  }
  std::printf("cpp tokens: %d checks OK\n", g_checks);
  return 0;
}
