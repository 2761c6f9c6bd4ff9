// C++ API check of the 8-bit paged cache and of choosing tokens (aurora_amd/csrc/aurora.hpp: PagedKvCache<uint8_t>,
// PagedKvAppendKernel, PagedKvReadKernel, PagedMhaKernel, SampleKernel), built with g++ against libaurora_hip.so.
//   e4m3_check        no device needed: the scratch's size, and refusals of a cache.
//   e4m3_check gpu    a sequence appended, read back and attended to, and tokens chosen, against plain loops.
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

int gpu_checks() {
  GpuContext ctx(0);
  const uint32_t H = 4, KV = 2, dh = 32, page = 16, S = 4, n = 21, d = H * dh, row = KV * dh;
  std::mt19937 g(1);
  std::normal_distribution<float> normal;
  auto make = [&](size_t len) {
    std::vector<float> v(len);
    for (auto& x : v) x = normal(g);
    return v;
  };
  auto i32 = [&](std::vector<int32_t> v) { return GpuBuffer<int32_t>::from_slice(ctx, v); };
  auto f32 = [&](const std::vector<float>& v) { return GpuBuffer<float>::from_slice(ctx, v); };
  aurora::PagedKvCache<uint8_t> cache(ctx, 3, page, KV, dh, S);
  auto off = i32({0, (int32_t)n}), len = i32({(int32_t)n}), pages = i32({2, 0});
  aurora::PagedBatch batch(off, len, pages, 1, 2, n, n, n);
  const auto q = make(n * d), k = make(n * row), v = make(n * row);
  auto table = GpuBuffer<float>::zeros(ctx, 1), qo = GpuBuffer<float>::zeros(ctx, n * d);
  aurora::PagedKvAppendKernel{}.dispatch_into(ctx, cache, batch, f32(q), f32(k), f32(v), qo, table, 0, 0, H);
  auto ko = GpuBuffer<float>::zeros(ctx, n * row), vo = GpuBuffer<float>::zeros(ctx, n * row);
  aurora::PagedKvReadKernel{}.dispatch_into(ctx, cache, batch, ko, vo, 0, n);
  const auto kr = ko.download(), vr = vo.download();
  for (uint32_t i = 0; i < n * row; ++i)  // half a step of e4m3, or of the smallest numbers of a scale for values below 7
    for (auto [x, y] : {std::pair<float, float>{k[i], kr[i]}, {v[i], vr[i]}})
      if (std::fabs(x - y) > std::fabs(x) / 16 + std::ldexp(1.f, -16)) return fail("read back", x - y);
  auto out = GpuBuffer<float>::zeros(ctx, n * d), lse = GpuBuffer<float>::zeros(ctx, n * H);
  GpuBuffer<float> ws(ctx, aurora::PagedMhaKernel::scratch_len(cache, batch, H) + 1);
  aurora::PagedMhaKernel{}.dispatch_into(ctx, cache, batch, qo, out, lse, ws, H);
  const auto got = out.download();
  double worst = 0;
  for (uint32_t i = 0; i < n; ++i)
    for (uint32_t h = 0; h < H; ++h) {
      const uint32_t hk = h / (H / KV);
      std::vector<double> sc(i + 1);
      double mx = -1e300, sum = 0;
      for (uint32_t j = 0; j <= i; ++j) {
        for (uint32_t c = 0; c < dh; ++c) sc[j] += (double)q[i * d + h * dh + c] * kr[j * row + hk * dh + c];
        mx = std::max(mx, sc[j] /= std::sqrt((double)dh));
      }
      for (auto& x : sc) sum += (x = std::exp(x - mx));
      for (uint32_t c = 0; c < dh; ++c) {
        double o = 0;
        for (uint32_t j = 0; j <= i; ++j) o += sc[j] / sum * vr[j * row + hk * dh + c];
        worst = std::max(worst, std::fabs(o - got[i * d + h * dh + c]));
      }
    }
  if (!(worst < 2.5e-5)) return fail("PagedMhaKernel", worst);

  // weights 1, 2, 4, 1: shares of an eighth, a fourth, a half and an eighth
  const float l2 = std::log(2.f);
  std::vector<float> logits;
  for (int r = 0; r < 4; ++r) logits.insert(logits.end(), {0.f, l2, 2 * l2, 0.f});
  auto tokens = GpuBuffer<int32_t>::zeros(ctx, 4);
  auto logprob = GpuBuffer<float>::zeros(ctx, 4);
  GpuBuffer<uint8_t> scratch(ctx, aurora::SampleKernel::scratch_len(4, 4) + 1);
  const auto x = f32(logits), u = f32({0.1f, 0.2f, 0.8f, 0.99f});
  aurora::SampleKernel{}.dispatch_into(ctx, x, u, tokens, logprob, scratch, 4, 4);
  auto t = tokens.download();
  if (t[0] != 0 || t[1] != 1 || t[2] != 2 || t[3] != 3) return fail("SampleKernel", t[0] * 1000 + t[1] * 100 + t[2] * 10 + t[3]);
  if (std::fabs(logprob.download()[2] + l2) > 1e-6) return fail("log-probability", logprob.download()[2]);
  const auto two = i32({2, 2, 2, 2});
  aurora::SampleKernel{}.dispatch_into(ctx, x, u, tokens, logprob, scratch, 4, 4, nullptr, &two);
  t = tokens.download();
  if (t[0] != 1 || t[1] != 1 || t[2] != 2 || t[3] != 2) return fail("top_k", t[0] * 1000 + t[1] * 100 + t[2] * 10 + t[3]);
  try {
    aurora::SampleKernel{}.dispatch_into(ctx, x, u, tokens, GpuBuffer<float>::zeros(ctx, 3), scratch, 4, 4);
    return fail("short buffer accepted", 0);
  } catch (const aurora::Error& e) {
    if (e.code != AUR_EINVAL) return fail("short buffer: code", e.code);
  }
  try {
    GpuBuffer<float> wide(ctx, 40000);
    aurora::SampleKernel{}.dispatch_into(ctx, wide, u, tokens, logprob, scratch, 1, 40000);
    return fail("short scratch accepted", 0);
  } catch (const aurora::Error& e) {
    if (e.code != AUR_EINVAL) return fail("short scratch: code", e.code);
  }
  std::printf("OK gpu: 8-bit append, read back and attention (largest error %.2g), choice of tokens\n", worst);
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
  uint8_t* const p = reinterpret_cast<uint8_t*>(0x10000);
  int32_t* const i = reinterpret_cast<int32_t*>(p);
  aur_paged_cache c{p, p, 64, 16, 2, 32, AUR_PAGED_E4M3, p, p, 16};
  const aur_paged_batch b{i, i, i, i, 4, 64, 4, 1, 1000, 300, 4096};
  if (aur_mha_paged_ws_bytes(&c, &b, 4) == 0) return fail("scratch of a valid batch", 0);
  c.scale_len = 32;
  if (aur_mha_paged_ws_bytes(&c, &b, 4) != 0 || !std::strstr(aur_last_error(nullptr), "scale_len")) return fail("scale_len", 0);
  if (aur_sample_ws_bytes(8, 32768) != 0 || aur_sample_ws_bytes(8, 32769) == 0) return fail("sampling scratch", 0);
  std::printf("OK no-gpu\n");
  return 0;
}
