// A block of experts through the C++ API (needs a GPU): routing, products and the way into the residual stream with w4::gpu,
// against arithmetic in 64 bits; refusals throw before any device work.
#include <cmath>
#include <random>
#include <vector>

#include "check.hpp"
#include "w4/gpu.hpp"
#include "w4/pack.hpp"

using namespace w4;
using namespace w4::gpu;

namespace {

template <class T>
struct Dev {
  T* p = nullptr;
  size_t n;
  explicit Dev(const std::vector<T>& host) : n(host.size()) {
    hip_check(hipMalloc((void**)&p, n * sizeof(T)), "hipMalloc");
    hip_check(hipMemcpy(p, host.data(), n * sizeof(T), hipMemcpyHostToDevice), "upload");
  }
  Dev(const Dev&) = delete;
  Dev& operator=(const Dev&) = delete;
  ~Dev() { (void)hipFree(p); }
  std::vector<T> get() const {
    std::vector<T> host(n);
    hip_check(hipDeviceSynchronize(), "sync");
    hip_check(hipMemcpy(host.data(), p, n * sizeof(T), hipMemcpyDeviceToHost), "download");
    return host;
  }
};

}  // namespace

int main() {
  Checks t;
  const int T = 5, E = 4, k = 2, K = 128, I = 32, P = T * k;
  std::mt19937_64 rng(1);
  std::normal_distribution<double> normal;
  std::vector<float> logits(T * E);
  for (auto& v : logits) v = (float)normal(rng);
  std::vector<double> w((size_t)E * 2 * I * K);
  for (auto& v : w) v = 0.05 * normal(rng);
  std::vector<__half> x(T * K);
  for (auto& v : x) v = __float2half((float)normal(rng));
  const PackedW packed = quantize(w, E * 2 * I, K, 32, true);

  const std::vector<float> pairs(P), stream(T * I);
  Dev<float> d_logits(logits), d_w(pairs), d_r(stream), d_r2(stream);
  Dev<int> d_ids((std::vector<int>(P))), d_order((std::vector<int>(P))), d_offsets((std::vector<int>(E + 1)));
  Dev<__half> d_x(x), d_y((std::vector<__half>((size_t)P * I))), d_h((std::vector<__half>(T * I)));
  Dev<__half> d_pre(std::vector<__half>(I, __float2half(1.f)));
  Dev<uint32_t> d_q(packed.q);
  Dev<__half> d_s(packed.scales);
  const DevicePackedW view{E * 2 * I, K, 32, K / 32, 1, d_q.p, d_s.p, nullptr};
  const Router router{E, k, 0, 1, 1, 1, 1, 1.f, nullptr};
  const size_t bytes = route_experts_workspace(router, T);
  Dev<char> space(std::vector<char>(bytes + 16));
  route_experts(router, d_logits.p, 0, T, nullptr, d_ids.p, d_w.p, d_order.p, d_offsets.p, space.p, bytes);
  const DeviceExpertRows rows{E, T, k, d_offsets.p, d_order.p};
  gemm_experts(view, rows, Act::silu, d_x.p, true, d_y.p, true);
  const DeviceBlockNorm norm{I, 0, 1e-6f, 1.f, nullptr, nullptr, nullptr, 0, d_pre.p, nullptr};
  residual_norm(norm, T, k, d_y.p, d_w.p, nullptr, d_r.p, d_r2.p, d_h.p);

  const auto ids = d_ids.get();
  const auto weights = d_w.get();
  const auto y = d_y.get();
  const auto r2 = d_r2.get();
  const auto h = d_h.get();
  const auto dq = dequant_all(packed);
  for (int i = 0; i < T; ++i) {
    int best = 0, next = -1;
    for (int e = 1; e < E; ++e)
      if (logits[i * E + e] > logits[i * E + best]) best = e;
    for (int e = 0; e < E; ++e)
      if (e != best && (next < 0 || logits[i * E + e] > logits[i * E + next])) next = e;
    t.expect(ids[2 * i] == best && ids[2 * i + 1] == next, "choices");
    const double a = 1.0 / (1.0 + std::exp((double)logits[i * E + next] - logits[i * E + best]));
    // two exponentials, a sum and a quotient of logits that are less than 8 apart
    t.expect(std::fabs(weights[2 * i] - a) < 32 * 0x1p-24 && std::fabs(weights[2 * i + 1] - (1 - a)) < 32 * 0x1p-24, "weights");
    double sq = 0;
    std::vector<double> sum(I, 0.0);
    for (int j = 0; j < k; ++j)
      for (int c = 0; c < I; ++c) {
        double g = 0, u = 0, ga = 0, ua = 0;
        const size_t row = (size_t)ids[2 * i + j] * 2 * I + c;
        for (int n = 0; n < K; ++n) {
          const double xg = (double)__half2float(x[i * K + n]) * (double)__half2float(dq[row * K + n]);
          const double xu = (double)__half2float(x[i * K + n]) * (double)__half2float(dq[(row + I) * K + n]);
          g += xg, u += xu, ga += std::fabs(xg), ua += std::fabs(xu);
        }
        const double act = g / (1 + std::exp(-g)), want = act * u, got = __half2float(y[(size_t)(2 * i + j) * I + c]);
        // FP32 sums of K terms, the gate's slope below 1.13, its arithmetic, one rounding to a half
        const double eps = (K + 8) * 0x1p-24;
        const double off = 1.13 * eps * ga * (std::fabs(u) + eps * ua) + std::fabs(act) * (eps * ua + (12 + std::fabs(g)) * 0x1p-23 * std::fabs(u));
        t.expect(std::fabs(got - want) <= off + 0x1p-11 * (std::fabs(want) + off) + 0x1p-25, "product");
        sum[c] += weights[2 * i + j] * got;
      }
    for (int c = 0; c < I; ++c) sq += sum[c] * sum[c];
    for (int c = 0; c < I; ++c) {
      const double want = sum[c] / std::sqrt(sq / I + 1e-6);
      // three FP32 steps a term; sums of squares in 64 steps, one rounding to a half
      t.expect(std::fabs(r2[i * I + c] - sum[c]) <= 8 * 0x1p-24 * std::sqrt(sq), "residual");
      t.expect(std::fabs((double)__half2float(h[i * I + c]) - want) <= (0x1p-11 + 64 * 0x1p-24) * std::fabs(want) + 8 * 0x1p-24 * std::sqrt(I) + 0x1p-25, "norm");
    }
  }
  t.throws_invalid([&] { gemm_experts(view, DeviceExpertRows{3, T, k, d_offsets.p, d_order.p}, Act::silu, d_x.p, true, d_y.p, true); },
                                  "N is no multiple of the experts");
  t.throws_invalid([&] { residual_norm(norm, T, 0, d_y.p, d_w.p, nullptr, d_r.p, d_r2.p, d_h.p); }, "no terms");
  return t.finish("experts");
}
