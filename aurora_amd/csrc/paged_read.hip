// Reading a paged K/V cache back as dense fp32 rows: key x of a sequence's axis
// (prefix, then its own keys) goes to row x − first of the sequence's `count`
// rows, whatever page it lies in; rows without a key become zeros.
//
// One thread moves 4 columns, so that a wave writes whole 1 KiB pieces of a row.
// Bound by HBM: an fp32 element is 4 bytes read and 4 written, one of e4m3 1 and 4.  32 sequences of 1280 keys,
// 16 heads of 64, in e4m3: 58 us, 6.5 TB/s (a large fill writes 6.9); with a row to a thread and stores that stay
// in the caches 103.
#include "common.hpp"
#include "paged.hpp"

using namespace aurpaged;

namespace {

struct ReadArgs {
  Batch b;
  const void *kp, *vp;
  float *k, *v;
  const uint8_t *ks, *vs;
  int ssh;
  int Hkv, dh, n_pages, sh, ld, first, count;
};

typedef unsigned uint2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ floatx4 get(const float* p, float) { return *reinterpret_cast<const floatx4*>(p); }
__device__ __forceinline__ floatx4 get(const __bf16* p, float) {
  const uint2v u = *reinterpret_cast<const uint2v*>(p);
  return floatx4{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
                 __uint_as_float(u[1] & 0xffff0000u)};
}
__device__ __forceinline__ floatx4 get(const e4m3* p, float scale) {
  const unsigned u = *reinterpret_cast<const unsigned*>(p);
  const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(u, scale, false);
  const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(u, scale, true);
  return floatx4{lo[0], lo[1], hi[0], hi[1]};
}

// A block has ROWS rows to a thread of one sequence, units of 4 columns of them; their pages' numbers, then their
// scales and elements, are under way together.
constexpr int ROWS = 4;
template <class T>
__global__ void __launch_bounds__(256) read_kernel(ReadArgs a, int lanes, int turns) {
  const int s = blockIdx.x / turns, d4 = a.Hkv * a.dh / 4;
  const int len = min(max(a.b.own_len[s], 0), a.b.max_own);
  const int u0 = threadIdx.x % lanes, per = 256 / lanes, lead = threadIdx.x / lanes;
  if (lead >= per) return;
  const int i0 = (blockIdx.x - s * turns) * ROWS * per + lead;
  int row[ROWS];  // in the pools, −1: no key
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int x = a.first + i0 + r * per, own = x - a.b.prefix_len;
    const bool is = i0 + r * per < a.count;
    row[r] = -1;
    if (is && own < 0)
      row[r] = a.b.prefix_pages[x >> a.sh];
    else if (is && own < len)
      row[r] = a.b.pages[(size_t)s * a.b.max_pages + (own >> a.sh)];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int x = a.first + i0 + r * per, own = x - a.b.prefix_len;
    row[r] = (unsigned)row[r] < (unsigned)a.n_pages ? (row[r] << a.sh) + ((own < 0 ? x : own) & ((1 << a.sh) - 1)) : -1;
  }
  for (int u = u0; u < d4; u += lanes) {
    const int head = sizeof(T) == 1 ? 4 * u / a.dh : 0;
    floatx4 k[ROWS], v[ROWS];
    float ks[ROWS], vs[ROWS];
    if (sizeof(T) == 1) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const size_t at = scale_index(max(row[r], 0), head, a.Hkv, a.sh, a.ssh);
        ks[r] = scale_of(a.ks[at]);
        vs[r] = scale_of(a.vs[at]);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {  // (where no key is, row 0's, and not written)
      const size_t from = (size_t)max(row[r], 0) * a.Hkv * a.dh + 4 * u;
      k[r] = v[r] = floatx4{0.f, 0.f, 0.f, 0.f};
      if (a.k) k[r] = get(static_cast<const T*>(a.kp) + from, ks[r]);
      if (a.v) v[r] = get(static_cast<const T*>(a.vp) + from, vs[r]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int i = i0 + r * per;
      if (i >= a.count) break;
      const size_t to = ((size_t)s * a.count + i) * a.ld + 4 * u;
      if (a.k) __builtin_nontemporal_store(row[r] < 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : k[r], reinterpret_cast<floatx4*>(a.k + to));
      if (a.v) __builtin_nontemporal_store(row[r] < 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : v[r], reinterpret_cast<floatx4*>(a.v + to));
    }
  }
}

}  // namespace

extern "C" int aur_kv_read_paged(aur_ctx* ctx, const aur_paged_cache* cache, const aur_paged_batch* batch, float* k_out,
                                 float* v_out, uint32_t ld, uint32_t first, uint32_t count) {
  AUR_CHECK_CTX(ctx);
  const char* who = "aur_kv_read_paged";
  ReadArgs a{};
  aur_paged_batch all{};  // what the checks look at: no new tokens
  if (batch) {
    all = *batch;
    all.n_tok = 0;
  }
  if (int rc = check_paged(ctx, who, cache, batch ? &all : nullptr, &a.b)) return rc;
  const uint32_t row = cache->n_kv_head * cache->d_head;
  if (a.b.b && (!a.b.own_len || (a.b.max_own && !a.b.pages) || (a.b.prefix_len && !a.b.prefix_pages)))
    return aur::set_error(ctx, AUR_EINVAL, "%s: null array in the batch", who);
  if (!aligned16(k_out) || !aligned16(v_out) || ld < row || ld % 4 || ld > 0x7fffffffu)
    return aur::set_error(ctx, AUR_EINVAL, "%s: ld=%u (a multiple of 4, at least %u), rows 16-byte aligned", who, ld, row);
  if ((uint64_t)first + count > (uint64_t)a.b.prefix_len + a.b.max_own)
    return aur::set_error(ctx, AUR_EINVAL, "%s: keys %u to %u of %d + %d", who, first, first + count, a.b.prefix_len,
                          a.b.max_own);
  if (a.b.b == 0 || count == 0 || (!k_out && !v_out)) return 0;
  a.kp = cache->k; a.vp = cache->v; a.k = k_out; a.v = v_out;
  a.Hkv = (int)cache->n_kv_head; a.dh = (int)cache->d_head; a.n_pages = (int)cache->n_pages;
  a.sh = log2_of(cache->page_len); a.ld = (int)ld; a.first = (int)first; a.count = (int)count;
  const int d4 = (int)row / 4, lanes = d4 < 256 ? d4 : 256, rows = ROWS * (256 / lanes);
  const int turns = ((int)count + rows - 1) / rows;
  if ((uint64_t)turns * a.b.b > kMaxBlocks)
    return aur::set_error(ctx, AUR_ELIMIT, "%s: %u keys of %d sequences", who, count, a.b.b);
  const dim3 grid((unsigned)(turns * a.b.b));
  if (cache->dtype == AUR_PAGED_F32) {
    hipLaunchKernelGGL(read_kernel<float>, grid, dim3(256), 0, ctx->stream, a, lanes, turns);
  } else if (cache->dtype == AUR_PAGED_BF16) {
    hipLaunchKernelGGL(read_kernel<__bf16>, grid, dim3(256), 0, ctx->stream, a, lanes, turns);
  } else {
    a.ks = cache->k_scale; a.vs = cache->v_scale; a.ssh = log2_of(cache->scale_len);
    hipLaunchKernelGGL(read_kernel<e4m3>, grid, dim3(256), 0, ctx->stream, a, lanes, turns);
  }
  AUR_LAUNCH_CHECK(ctx, "read_kernel");
  return 0;
}
