// C++ API check of the paged K/V cache (aurora_amd/csrc/aurora.hpp: PagedKvCache, PagedBatch,
// RotaryTableKernel, PagedKvAppendKernel, PagedMhaKernel), built with g++ against libaurora_hip.so.
//   paged_check        no device needed: the scratch's size, and refusals of a batch.
//   paged_check gpu    a prefix and two sequences, appended and attended to, against plain loops in double.
// Exit status 0 on success; the failing check is printed.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "../../aurora_amd/csrc/aurora.hpp"

using aurora::GpuBuffer;
using aurora::GpuContext;

namespace {

int fail(const char* what, double v) {
  std::printf("FAIL %s (%g)\n", what, v);
  return 1;
}

// x [n, H, dh] turned by the angles of positions pos0 …, columns (u, u + rot/2) of a head as a pair.
std::vector<double> turned(const std::vector<float>& x, uint32_t n, uint32_t H, uint32_t dh, uint32_t rot, uint32_t pos0) {
  std::vector<double> y(x.begin(), x.begin() + (size_t)n * H * dh);
  for (uint32_t i = 0; i < n; ++i)
    for (uint32_t h = 0; h < H; ++h)
      for (uint32_t u = 0; u < rot / 2; ++u) {
        const double a = (pos0 + i) * std::pow(10000.0, -2.0 * u / rot);
        double* p = &y[((size_t)i * H + h) * dh];
        const double p0 = p[u], p1 = p[u + rot / 2];
        p[u] = p0 * std::cos(a) - p1 * std::sin(a);
        p[u + rot / 2] = p1 * std::cos(a) + p0 * std::sin(a);
      }
  return y;
}

int gpu_checks() {
  GpuContext ctx(0);
  const uint32_t H = 4, KV = 2, dh = 32, rot = 32, page = 8, P = 13, n0 = 5, n1 = 9, n = n0 + n1, d = H * dh, row = KV * dh;
  std::mt19937 g(1);
  std::uniform_real_distribution<float> u(-1.f, 1.f);
  auto make = [&](size_t len) {
    std::vector<float> v(len);
    for (auto& x : v) x = u(g);
    return v;
  };
  auto i32 = [&](std::vector<int32_t> v) { return GpuBuffer<int32_t>::from_slice(ctx, v); };
  auto f32 = [&](const std::vector<float>& v) { return GpuBuffer<float>::from_slice(ctx, v); };
  aurora::PagedKvCache<float> cache(ctx, 6, page, KV, dh);
  auto table = GpuBuffer<float>::zeros(ctx, 32 * rot);
  aurora::RotaryTableKernel{}.dispatch_into(ctx, table, 32, rot);
  aurora::PagedKvAppendKernel append;
  aurora::PagedMhaKernel mha;

  // the prefix, a batch of one sequence in pages 4 and 1
  auto pq = make(P * d), pk = make(P * row), pv = make(P * row);
  auto prefix = i32({4, 1}), off0 = i32({0, (int32_t)P}), len0 = i32({(int32_t)P});
  aurora::PagedBatch b0(off0, len0, prefix, 1, 2, P, P, P);
  auto qo0 = GpuBuffer<float>::zeros(ctx, P * d);
  append.dispatch_into(ctx, cache, b0, f32(pq), f32(pk), f32(pv), qo0, table, 32, rot, H);

  // two sequences behind it
  auto q = make(n * d), k = make(n * row), v = make(n * row);
  auto off = i32({0, (int32_t)n0, (int32_t)n}), len = i32({(int32_t)n0, (int32_t)n1}), pages = i32({5, -1, 0, 3});
  aurora::PagedBatch b1(off, len, pages, 2, 2, n, n1, n1);
  b1.behind(prefix, P);
  auto qo = GpuBuffer<float>::zeros(ctx, n * d), out = GpuBuffer<float>::zeros(ctx, n * d), lse = GpuBuffer<float>::zeros(ctx, n * H);
  append.dispatch_into(ctx, cache, b1, f32(q), f32(k), f32(v), qo, table, 32, rot, H);
  GpuBuffer<float> ws(ctx, aurora::PagedMhaKernel::scratch_len(cache, b1, H) + 1);
  mha.dispatch_into(ctx, cache, b1, qo, out, lse, ws, H);
  const auto got = out.download();

  const auto tpk = turned(pk, P, KV, dh, rot, 0);
  double worst = 0;
  for (uint32_t s = 0; s < 2; ++s) {
    const uint32_t lo = s ? n0 : 0, cnt = s ? n1 : n0;
    const std::vector<float> ks(k.begin() + lo * row, k.end()), qs(q.begin() + lo * d, q.end());
    const auto tk = turned(ks, cnt, KV, dh, rot, P), tq = turned(qs, cnt, H, dh, rot, P);
    for (uint32_t i = 0; i < cnt; ++i)
      for (uint32_t h = 0; h < H; ++h) {
        const uint32_t hk = h / (H / KV), keys = P + i + 1;
        auto at = [&](const std::vector<double>& pre, const std::vector<double>& own, uint32_t j, uint32_t c) {
          return j < P ? pre[(j * KV + hk) * dh + c] : own[((j - P) * KV + hk) * dh + c];
        };
        const std::vector<double> pvd(pv.begin(), pv.end()), vd(v.begin() + lo * row, v.end());
        std::vector<double> sc(keys);
        double mx = -1e300, sum = 0;
        for (uint32_t j = 0; j < keys; ++j) {
          for (uint32_t c = 0; c < dh; ++c) sc[j] += tq[(i * H + h) * dh + c] * at(tpk, tk, j, c);
          mx = std::max(mx, sc[j] /= std::sqrt((double)dh));
        }
        for (auto& x : sc) sum += (x = std::exp(x - mx));
        for (uint32_t c = 0; c < dh; ++c) {
          double o = 0;
          for (uint32_t j = 0; j < keys; ++j) o += sc[j] / sum * at(pvd, vd, j, c);
          worst = std::max(worst, std::fabs(o - got[((lo + i) * H + h) * dh + c]));
        }
      }
  }
  // scores of 32 products below 1: off by (32 + 4)·2^-24·32/√32 at most, twice, and 22 keys' sums
  if (!(worst < 2.5e-5)) return fail("PagedMhaKernel", worst);
  try {
    mha.dispatch_into(ctx, cache, b1, qo, GpuBuffer<float>::zeros(ctx, n * d - 1), lse, ws, H);
    return fail("short output buffer accepted", 0);
  } catch (const aurora::Error& e) {
    if (e.code != AUR_EINVAL) return fail("short output buffer: code", e.code);
  }
  std::printf("OK gpu: paged append and attention (largest error %.2g)\n", worst);
  return 0;
}

}  // namespace

int main(int argc, char** argv) {
  if (argc > 1 && std::strcmp(argv[1], "gpu") == 0) {
    try {
      return gpu_checks();
    } catch (const aurora::Error& e) {
      std::printf("FAIL aurora::Error %d: %s\n", e.code, e.what());
      return 1;
    }
  }
  void* const p = reinterpret_cast<void*>(0x10000);
  int32_t* const i = static_cast<int32_t*>(p);
  const aur_paged_cache c{p, p, 64, 16, 2, 32, AUR_PAGED_F32};
  aur_paged_batch b{i, i, i, i, 4, 64, 4, 1, 1000, 300, 4096};
  if (aur_mha_paged_ws_bytes(&c, &b, 4) == 0) return fail("scratch of a valid batch", 0);
  b.max_own = 64 * 16 + 1;
  if (aur_mha_paged_ws_bytes(&c, &b, 4) != 0 || !std::strstr(aur_last_error(nullptr), "max_own")) return fail("max_own", 0);
  std::printf("OK no-gpu\n");
  return 0;
}
