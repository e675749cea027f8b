// Serving over a paged FP8 cache through the C++ API (needs a GPU): a prompt and decode steps planned, written and
// attended with w4::gpu, against arithmetic in 64 bits on what the cache holds.
#include <cmath>
#include <random>
#include <vector>

#include "check.hpp"
#include "w4/gpu.hpp"

using namespace w4;
using namespace w4::gpu;

namespace {

template <class T>
struct Dev {
  T* p = nullptr;
  size_t n;
  explicit Dev(const std::vector<T>& host) : n(host.size()) {
    hip_check(hipMalloc((void**)&p, n * sizeof(T)), "hipMalloc");
    put(host);
  }
  Dev(const Dev&) = delete;
  Dev& operator=(const Dev&) = delete;
  ~Dev() { (void)hipFree(p); }
  void put(const std::vector<T>& host) { hip_check(hipMemcpy(p, host.data(), host.size() * sizeof(T), hipMemcpyHostToDevice), "upload"); }
  std::vector<T> get() const {
    std::vector<T> host(n);
    hip_check(hipDeviceSynchronize(), "sync");
    hip_check(hipMemcpy(host.data(), p, n * sizeof(T), hipMemcpyDeviceToHost), "download");
    return host;
  }
};

double value(uint8_t b) {
  const int e = (b >> 3) & 15, m = b & 7;
  const double v = e ? (8 + m) * std::ldexp(1.0, e - 10) : m * std::ldexp(1.0, -9);
  return b & 0x80 ? -v : v;
}

}  // namespace

int main() {
  Checks t;
  const int H = 2, group = 4, D = 64, page = 16, npages = 24, nseq = 3, R = 6, places = 48;
  const size_t row = (size_t)H * D, qrow = row * group;
  std::mt19937_64 rng(1);
  std::normal_distribution<double> normal;
  auto halves = [&](size_t n) {
    std::vector<__half> x(n);
    for (auto& h : x) h = __float2half_rn((float)normal(rng));
    return x;
  };
  Dev<uint8_t> qk(std::vector<uint8_t>((size_t)H * npages * page * D, 0x7F)), qv(std::vector<uint8_t>(qk.n, 0x7F));
  Dev<__half> sk(std::vector<__half>((size_t)H * npages)), sv(std::vector<__half>((size_t)H * npages));
  const std::vector<int> none(places);
  Dev<int> bt(std::vector<int>(nseq * R, -1)), lens(none), cu(none), cached(none), added(none), slots(none), positions(none),
      result(none), status(none);
  std::vector<int> pages(npages);
  for (int i = 0; i < npages; ++i) pages[i] = (7 * i + 3) % npages;
  Dev<int> free_pages(pages), range(std::vector<int>{0, npages});
  const DeviceF8Pages view{H, D, page, npages, qk.p, sk.p, qv.p, sv.p};
  const DevicePagedBatch batch{nseq, places, places, R * page, R, bt.p, lens.p, cu.p};
  Dev<uint8_t> space(std::vector<uint8_t>(attention_f8_pages_workspace(view, batch, group) + 16, 0));
  Dev<__half> out(std::vector<__half>(places * qrow));
  std::vector<int> have(nseq, 0);
  std::vector<std::vector<double>> keys[2];  // what was given, in order, per sequence
  keys[0].resize(nseq), keys[1].resize(nseq);
  int taken = 0;
  const std::vector<std::vector<int>> steps{{20, 1, 16}, {1, 1, 1}, {1, 5, 0}, {1, 1, 1}};
  for (const auto& more : steps) {
    const auto q = halves(places * qrow), k = halves(places * row), v = halves(places * row);
    Dev<__half> q_d(q), k_d(k), v_d(v);
    cached.put(have), added.put(more), range.put({taken, npages});
    paged_tables(batch, page, npages, cached.p, added.p, free_pages.p, range.p, slots.p, positions.p, result.p);
    quantize_f8_pages_async(view, k_d.p, v_d.p, 0, slots.p, places, status.p);
    attention_f8_pages(view, batch, group, true, q_d.p, 0, out.p, space.p, space.n);
    const auto got = out.get();
    const auto r = result.get(), table = bt.get();
    t.expect(r[1] == 0 && status.get()[0] == 0, "a step's status");
    taken += r[0];
    const std::vector<uint8_t> codes[2] = {qk.get(), qv.get()};
    const std::vector<__half> scales[2] = {sk.get(), sv.get()};
    int first = 0;
    for (int s = 0; s < nseq; ++s) {
      for (int i = 0; i < more[s]; ++i)
        for (size_t e = 0; e < row; ++e) {
          keys[0][s].push_back(__half2float(k[(first + i) * row + e]));
          keys[1][s].push_back(__half2float(v[(first + i) * row + e]));
        }
      have[s] += more[s];
      const int L = have[s];
      bool written = true, attended = true;
      auto at = [&](int side, int h, int p, int d) {
        const size_t pg = (size_t)h * npages + table[s * R + p / page];
        return value(codes[side][(pg * page + p % page) * D + d]) * (double)__half2float(scales[side][pg]);
      };
      // half a step of E4M3, and of its subnormals once for each time a scale was raised (at most three here)
      for (int side = 0; side < 2; ++side)
        for (int p = 0; p < L; ++p)
          for (int h = 0; h < H; ++h)
            for (int d = 0; d < D; ++d) {
              const double x = keys[side][s][p * row + h * D + d];
              const double sc = __half2float(scales[side][(size_t)h * npages + table[s * R + p / page]]);
              written = written && std::abs(at(side, h, p, d) - x) <= std::abs(x) / 16 + 4 * std::ldexp(sc, -10);
            }
      for (int i = 0; i < more[s]; ++i)
        for (int hq = 0; hq < H * group; ++hq) {
          const int h = hq / group, sees = L - more[s] + i + 1;
          std::vector<double> w(sees);
          double top = -1e300, sum = 0, rough = 0;
          for (int p = 0; p < sees; ++p) {
            double dot = 0, size = 0;
            for (int d = 0; d < D; ++d) {
              const double x = at(0, h, p, d) * __half2float(q[(first + i) * qrow + hq * D + d]);
              dot += x, size += std::abs(x);
            }
            w[p] = dot / std::sqrt((double)D), top = std::max(top, w[p]), rough = std::max(rough, size / std::sqrt((double)D));
          }
          const double most = std::abs(top);
          for (double& x : w) x = std::exp(x - top), sum += x;
          for (int d = 0; d < D; ++d) {
            double o = 0, a = 0, m = 0;
            for (int p = 0; p < sees; ++p) {
              const double z = at(1, h, p, d);
              o += w[p] / sum * z, a += w[p] / sum * std::abs(z), m += std::abs(z);
            }
            // weights and output rounded to halves; FP32 scores of D products, exponents and sums
            const double eps = (D + 4) * 0x1p-24 * rough + 0x1p-21 * (most + rough + 48) + sees * 0x1p-24;
            const double tol = 0x1p-11 * (a + std::abs(o)) + 2 * eps * a + 0x1p-25 * (1 + m);
            attended = attended && std::abs(__half2float(got[(first + i) * qrow + hq * D + d]) - o) <= tol;
          }
        }
      t.expect(written, "the cache holds the tokens");
      t.expect(attended, "attention over the cache");
      first += more[s];
    }
  }
  t.throws_invalid([&] { attention_f8_pages(view, batch, group, true, out.p, 0, out.p, space.p, 16); }, "workspace too small");
  t.throws_invalid([&] { attention_f8_pages_workspace(view, batch, 65); }, "query group");
  t.throws_invalid([&] { quantize_f8_pages_async(view, out.p, nullptr, 0, slots.p, 1, status.p); }, "null V");
  t.throws_invalid([&] { paged_tables(batch, 0, npages, cached.p, added.p, free_pages.p, range.p, slots.p, positions.p, result.p); },
                   "page of no rows");
  return t.finish("pages");
}
