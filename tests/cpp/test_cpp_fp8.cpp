// Routing to experts and the 8-bit floating-point products through the C++ host
// API (include/cascadia_int4.hpp), against plain loops in double over codes that
// need no rounding: one-hot rows and powers of two, whose results are exact.
//
// Prints one line per check and "cpp fp8: N checks OK"; exit status 1 on the first
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

// e4m3 code of 1, 2, 4, 8 (sign apart): exponent bias 7, 3 mantissa bits
uint8_t power(int e) { return (uint8_t)((7 + e) << 3); }
uint16_t bf16(float v) { return ci::f32_to_bf16_bits(v); }

}  // namespace

int main() {
  {  // routing: four experts, two tokens, ties to the lower id
    const std::vector<float> logits = {0.f, 2.f, 2.f, -1.f, 3.f, 0.f, 1.f, 3.f};
    const auto l = on_device(logits);
    ci::DeviceBuffer<int32_t> ids(4);
    ci::DeviceBuffer<float> w(4);
    ci::Router r{4, 2, CASCADIA_INT4_SCORE_SOFTMAX, 1, 1, 1, 1, 1.0f, nullptr};
    ci::route_experts(r, ci::DeviceSlice<const float>(l), ids, w);
    expect(ids.download() == std::vector<int32_t>({1, 2, 0, 3}), "route: ids");
    for (float v : w.download()) expect(std::fabs(v - 0.5f) < 1e-6f, "route: weights");
    std::vector<uint16_t> lb;
    for (float v : logits) lb.push_back(bf16(v));
    const auto b = on_device(lb);
    ci::route_experts(r, ci::DeviceSlice<const uint16_t>(b), ids, w);
    expect(ids.download() == std::vector<int32_t>({1, 2, 0, 3}), "route: bf16 logits");
    expect(refused([&] { ci::route_experts(r, ci::DeviceSlice<const float>(l), {ids.data(), 3}, w); }),
           "route: wrong length refused");
    r.n_groups = 3;
    expect(refused([&] { ci::route_experts(r, ci::DeviceSlice<const float>(l), ids, w); }),
           "route: groups that do not divide refused");
  }
  const size_t n = 144, k = 272, m = 5;  // two blocks each way and a short third of K
  std::vector<uint16_t> wb(n * k);
  for (size_t i = 0; i < wb.size(); ++i) wb[i] = bf16((float)(1 << (i * 7 % 4)) * (i % 3 ? 1.f : -1.f));
  const auto weights = on_device(wb);
  const auto q = ci::quantize_fp8_blocks(weights, n, k);
  {  // every block's largest is 8: scale 8 / 448, codes of powers of two times 56
    bool ok = true;
    for (float s : q.second.download()) ok = ok && s == 8.0f / 448.0f;
    expect(ok && q.second.size() == 2 * 3, "quantize_fp8_blocks: scales");
  }
  std::vector<float> x(m * k, 0.f);
  for (size_t t = 0; t < m; ++t) x[t * k + 61 * t] = 448.f;  // one-hot rows: code 448, scale 1
  const auto xd = on_device(x);
  ci::DeviceBuffer<uint8_t> xc(m * k);
  ci::DeviceBuffer<float> xs(m * 3);
  ci::quantize_fp8(ci::DeviceSlice<const float>(xd), m, k, xc, xs);
  ci::DeviceBuffer<float> y(m * n), y2(m * n);
  ci::fp8_gemm(q.first, q.second, ci::DeviceSlice<const float>(xd), n, k, m, y);
  ci::fp8_gemm(q.first, q.second,
               ci::Fp8Rows(ci::DeviceSlice<const uint8_t>(xc), ci::DeviceSlice<const float>(xs)), n,
               k, m, y2);
  {
    bool ok = true;
    const auto a = y.download(), b = y2.download();
    for (size_t t = 0; t < m; ++t)
      for (size_t r = 0; r < n; ++r) {
        const double want = 448.0 * ci::bf16_bits_to_f32(wb[r * k + 61 * t]);
        ok = ok && std::fabs(a[t * n + r] - want) <= 1e-6 * std::fabs(want) &&
             a[t * n + r] == b[t * n + r];
      }
    expect(ok, "fp8_gemm: f32 rows and codes");
  }
  expect(refused([&] { ci::fp8_gemm(q.first, q.second, ci::DeviceSlice<const float>(xd), n, k, m + 1, y); }),
         "fp8_gemm: wrong length refused");
  {  // one expert per token: silu(g) u with g = u = 8, through a unit down row
    const size_t e = 3, h = 32, i = 16, t = 2;
    std::vector<uint8_t> gu(e * 2 * i * h, 0), dn(e * h * i, 0);
    for (size_t a = 0; a < e; ++a) {
      for (size_t j = 0; j < 2; ++j) gu[((a * 2 + j) * i + a) * h] = power((int)a);  // column 0
      dn[(a * h + 5) * i + a] = power(0);
    }
    const std::vector<float> gus(e * 2, 1.f / 448.f), dns(e, 1.f);
    const auto g = on_device(gu), d = on_device(dn);
    const auto gs = on_device(gus), ds = on_device(dns);
    const ci::Fp8Experts ex(g, gs, d, ds, e, h, i);
    std::vector<float> in(t * h, 0.f), res(t * h, 1.f);
    in[0] = in[h] = 448.f;  // code 448, scale 1: g = u = 2^a
    const auto xin = on_device(in), rin = on_device(res);
    const auto ids = on_device(std::vector<int32_t>{2, 0, 1, -1});
    const auto w = on_device(std::vector<float>{0.5f, 0.25f, 1.f, 1.f});
    ci::DeviceBuffer<float> out(t * h);
    ci::fp8_moe_forward(ex, ci::DeviceSlice<const float>(xin), ids, w, 2, out.slice(),
                        ci::DeviceSlice<const float>(rin));
    auto act = [](double v) { return v / (1 + std::exp(-v)) * v; };
    const auto o = out.download();
    // (bf16 slots: 2^-8 of each)
    const double a = 0.5 * act(4) + 0.25 * act(1), b = act(2);
    expect(std::fabs(o[5] - 1 - a) <= a / 256 && std::fabs(o[h + 5] - 1 - b) <= b / 256,
           "fp8_moe_forward: chosen experts");
    bool ok = true;
    for (size_t c = 0; c < t * h; ++c) ok = ok && (c % h == 5 || o[c] == 1.f);
    expect(ok, "fp8_moe_forward: the other columns are the residual");
    expect(refused([&] {
             ci::fp8_moe_forward(ex, ci::DeviceSlice<const float>(xin), ids, w, 3, out.slice());
           }),
           "fp8_moe_forward: wrong length refused");
    expect(refused([&] { ci::Fp8Experts bad(g, gs, d, ds, e, h, i + 8); }),
           "Fp8Experts: wrong dimensions refused");
  }
  std::printf("cpp fp8: %d checks OK\n", g_checks);
  return 0;
}
