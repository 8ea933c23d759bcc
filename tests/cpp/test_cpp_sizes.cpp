// Workspace sizes of the C++ host API (include/cascadia_int4.hpp) for sizes past 32 bits:
// refused, not cut off.  Without an argument host code alone; with one, also those of the
// layers that lay out weights on the device.
//
// Prints one line per check and "cpp sizes: N checks OK"; exit status 1 on the first
// failure.
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

template <class F>
bool refused(F f) {
  try {
    f();
  } catch (const std::invalid_argument &) {
    return true;
  }
  return false;
}

const size_t kPast = (size_t)1 << 32;

// workspace(top_k, n_tokens)
template <class F>
void check(const std::string &what, F workspace) {
  expect(workspace(2, 40) > 0, what + ": a size");
  expect(refused([&] { workspace(2, kPast + 40); }), what + ": n_tokens past 32 bits refused");
  expect(refused([&] { workspace(kPast + 2, 40); }), what + ": top_k past 32 bits refused");
}

}  // namespace

int main(int argc, char **) {
  {
    const size_t e = 2, r = 8, n = 16, k = 32;
    const uint16_t *p = reinterpret_cast<const uint16_t *>(size_t{1} << 20);  // (never read)
    const ci::Adapters a(ci::DeviceSlice<const uint16_t>(p, e * r * k),
                         ci::DeviceSlice<const uint16_t>(p, e * n * r), e, r, n, k);
    expect(a.workspace_bytes(40) > 0, "Adapters: a size");
    expect(refused([&] { a.workspace_bytes(kPast + 40); }), "Adapters: n_tokens past 32 bits refused");
    check("sort_tokens", [](size_t top_k, size_t t) {
      return ci::sort_tokens_workspace_bytes(t * 500, top_k, 384);
    });
  }
  if (argc > 1) {
    const size_t e = 2, h = 128, i = 128, flat = cascadia_int4_expert_bytes(h, i, 32);
    const std::vector<uint8_t> zeros(e * flat);
    const auto stack = ci::ExpertStack::upload(zeros.data(), e, h, i);
    const ci::MoeLayer layer(stack);
    check("MoeLayer", [&](size_t top_k, size_t t) { return layer.workspace_bytes(top_k, t); });

    ci::DeviceBuffer<uint8_t> gu(2 * e * i * h), down(e * h * i);
    ci::DeviceBuffer<float> gus(2 * e), ds(e);
    const std::vector<uint8_t> codes(2 * e * i * h);
    gu.upload(codes.data());
    down.upload(codes.data());
    const ci::Fp8Experts fp8(gu, gus, down, ds, e, h, i);
    check("Fp8Experts", [&](size_t top_k, size_t t) { return fp8.workspace_bytes(top_k, t); });
  }
  std::printf("cpp sizes: %d checks OK\n", g_checks);
  return 0;
}
