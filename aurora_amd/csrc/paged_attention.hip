// The entry points of the paged attention, and the join of a call's records; the items' kernels, what they
// compute and why, are in paged_attention.hpp.
#include "paged_attention.hpp"

namespace {

// out and lse of a row from the records of its ranges: one wave a row.  The lanes of a group have 4
// columns each, the groups take the ranges in turn and are added as a tree, so the order is fixed.
// Which ranges were written depends on the sequence's length; the loads do not wait for it (what lies in
// a range that was not is masked).  Of up to six dependent loads three remain: 7.2 → 4.7 µs for 16 rows of 17
// ranges, 3.8 → 3.0 µs for 512 rows of 2, 16 → 13 µs for 25,000 rows of 5.
// JOIN: ranges of a group that are under way at once.
template <int JOIN>
__global__ void __launch_bounds__(256) paged_join_kernel(MhaArgs a, int lanes) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int t = (int)(row / a.H), h = (int)(row - (long long)t * a.H);
  if (t >= a.b.n_tok) return;
  const int all = a.p_splits + a.o_splits, c = 4 * (lane % lanes), groups = 64 / lanes, g = lane / lanes;
  const size_t step = (size_t)a.b.n_tok * a.H, rec = (size_t)t * a.H + h;
  const float* ml = a.part_ml + 2 * rec;
  const float* o = a.part_o + rec * a.dh + min(c, a.dh - 4);
  auto pair = [&](int p) { return *reinterpret_cast<const float2v*>(ml + 2 * (size_t)min(p, all - 1) * step); };
  floatx4 v[JOIN];
  float2v w[JOIN];
#pragma unroll
  for (int i = 0; i < JOIN; ++i) {
    v[i] = load4(o + (size_t)min(g + i * groups, all - 1) * step * a.dh);
    w[i] = pair(g + i * groups);
  }
  const float2v first = pair(lane);
  int s = 0;
  for (int i0 = 0; i0 < a.b.b; i0 += 64) {
    const int i = i0 + lane;
    s += __popcll(__ballot(i < a.b.b && a.b.tok_off[i + 1] <= t));
  }
  if (s >= a.b.b) return;  // a row behind the last sequence
  const Seq q = sequence(a.b, s);
  if (t < q.lo || t - q.lo >= q.n) return;
  const int axis = q.len + (a.pooled ? 0 : a.b.prefix_len);
  const int np = a.p_splits + max((axis + a.o_keys - 1) / a.o_keys, 1);  // range 0 is always written
  float M = lane < np ? first[0] : -INFINITY;
  for (int p = lane + 64; p < np; p += 64) M = fmaxf(M, pair(p)[0]);
#pragma unroll
  for (int i = 1; i < 64; i *= 2) M = fmaxf(M, __shfl_xor(M, i, 64));
  auto factor = [&](float m) { return M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - M); };
  float L = lane < np ? factor(first[0]) * first[1] : 0.f;
  for (int p = lane + 64; p < np; p += 64) {
    const float2v x = pair(p);
    L += factor(x[0]) * x[1];
  }
#pragma unroll
  for (int i = 1; i < 64; i *= 2) L += __shfl_xor(L, i, 64);
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < JOIN; ++i)
    if (g + i * groups < np) sum += v[i] * factor(w[i][0]);
  for (int p = g + JOIN * groups; p < np; p += groups) sum += load4(o + (size_t)p * step * a.dh) * factor(pair(p)[0]);
#pragma unroll
  for (int i = 1; i < 64; i *= 2) {
    if (i < lanes) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], i, 64);
  }
  if (lane < lanes && c < a.dh)
    *reinterpret_cast<floatx4*>(a.out + (size_t)t * a.ld_o + (size_t)h * a.dh + c) =
        L == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : sum * (1.f / L);
  if (lane == 0 && a.lse) a.lse[(size_t)t * a.H + h] = L == 0.f ? -INFINITY : (M + __log2f(L)) * LN2;
}

constexpr uint32_t kMaxRows = 0x7fffff00u;  // query rows of a call, and a tile more, are ints

size_t ws_floats(const Plan& p, const Batch& b, int H, int dh) {
  return p.parts() > 1 ? (size_t)p.parts() * b.n_tok * H * (dh + 2) : 0;
}

Sizes sizes_of(const Batch& b, const aur_paged_cache& c, uint32_t n_head) {
  return {b.b, b.n_tok, b.max_tok, b.max_own, b.prefix_len, (int)c.n_kv_head, (int)(n_head / c.n_kv_head), (int)c.d_head,
          c.dtype == AUR_PAGED_F32, c.dtype == AUR_PAGED_E4M3};
}

void launch_items(const MhaArgs& a, const Sizes& z, int p_tile, int tile, unsigned items, hipStream_t st) {
  (z.f32 ? launch_items_f32 : z.e4m3 ? launch_items_e4m3 : launch_items_bf16)(a, z, p_tile, tile, items, st);
}

}  // namespace

extern "C" {

size_t aur_mha_paged_ws_bytes(const aur_paged_cache* cache, const aur_paged_batch* batch, uint32_t n_head) {
  Batch b;
  if (check_paged(nullptr, "aur_mha_paged_ws_bytes", cache, batch, &b) != 0 || n_head == 0 || n_head > 4096 ||
      (uint64_t)b.n_tok * n_head > kMaxRows || n_head % cache->n_kv_head != 0 || b.b == 0 || b.n_tok == 0)
    return 0;
  return 4 * ws_floats(make_plan(sizes_of(b, *cache, n_head)), b, (int)n_head, (int)cache->d_head);
}

int aur_mha_paged(aur_ctx* ctx, const aur_paged_cache* cache, const aur_paged_batch* batch, const float* q,
                  uint32_t ld_q, float* out, uint32_t ld_o, float* lse, float* scratch, size_t scratch_bytes,
                  uint32_t n_head) {
  AUR_CHECK_CTX(ctx);
  const char* who = "aur_mha_paged";
  MhaArgs a{};
  if (int rc = check_paged(ctx, who, cache, batch, &a.b)) return rc;
  if (n_head == 0 || n_head % cache->n_kv_head != 0)
    return aur::set_error(ctx, AUR_EINVAL, "%s: n_head=%u, a multiple of n_kv_head=%u", who, n_head, cache->n_kv_head);
  if (n_head > 4096 || (uint64_t)a.b.n_tok * n_head > kMaxRows)
    return aur::set_error(ctx, AUR_ELIMIT, "%s: n_tok=%d n_head=%u", who, a.b.n_tok, n_head);
  if (a.b.b == 0 || a.b.n_tok == 0) return 0;
  const uint32_t d = n_head * cache->d_head;
  if (!q || !out || !aligned16(q) || !aligned16(out))
    return aur::set_error(ctx, AUR_EINVAL, "%s: q and out must be there and 16-byte aligned", who);
  if (ld_q < d || ld_o < d || ld_q % 4 || ld_o % 4 || ld_q > 0x7fffffffu || ld_o > 0x7fffffffu)
    return aur::set_error(ctx, AUR_EINVAL, "%s: ld_q=%u ld_o=%u (multiples of 4, at least %u)", who, ld_q, ld_o, d);
  a.q = q; a.out = out; a.lse = lse; a.k = cache->k; a.v = cache->v;
  a.ld_q = (int)ld_q; a.ld_o = (int)ld_o;
  a.H = (int)n_head; a.Hkv = (int)cache->n_kv_head; a.G = a.H / a.Hkv; a.dh = (int)cache->d_head;
  a.n_pages = (int)cache->n_pages; a.sh = log2_of(cache->page_len);
  a.scale = 1.0f / sqrtf((float)a.dh);
  if (cache->dtype == AUR_PAGED_E4M3) {
    a.k_scale = cache->k_scale; a.v_scale = cache->v_scale; a.ssh = log2_of(cache->scale_len);
  }
  const Sizes z = sizes_of(a.b, *cache, n_head);
  const Plan p = make_plan(z);
  a.pooled = p.pooled;
  a.p_tiles = p.p_tiles; a.p_splits = p.p_splits; a.p_keys = p.p_keys;
  a.o_tiles = p.o_tiles; a.o_splits = p.o_splits; a.o_keys = p.o_keys;
  const size_t floats = ws_floats(p, a.b, a.H, a.dh);
  if (floats) {
    if (!scratch || !aligned16(scratch) || scratch_bytes < 4 * floats)
      return aur::set_error(ctx, AUR_EINVAL, "%s: scratch of %zu bytes (16-byte aligned), %zu needed", who,
                            scratch ? scratch_bytes : (size_t)0, 4 * floats);
    a.part_o = scratch;
    a.part_ml = scratch + (size_t)p.parts() * a.b.n_tok * a.H * a.dh;
  }
  const uint64_t p_groups = (uint64_t)p.p_tiles * p.p_splits, o_groups = (uint64_t)p.o_tiles * a.b.b * p.o_splits;
  a.by_xcd = cache->dtype == AUR_PAGED_E4M3 && heads_by_xcd(a.dh, p_groups, o_groups);
  const uint64_t p_items = items_of(a.by_xcd, p_groups, a.Hkv), o_items = items_of(a.by_xcd, o_groups, a.Hkv);
  const uint64_t rows4 = ((uint64_t)a.b.n_tok * n_head + 3) / 4;  // blocks of the join
  if (p_items + o_items > kMaxBlocks / 2 || rows4 > kMaxBlocks)
    return aur::set_error(ctx, AUR_ELIMIT, "%s: %llu + %llu blocks", who, (unsigned long long)p_items,
                          (unsigned long long)o_items);
  if (p.pooled && !p.together()) {
    a.p_items = (int)p_items;
    launch_items(a, z, 0, p.p_tile, (unsigned)p_items, ctx->stream);
    AUR_LAUNCH_CHECK(ctx, "paged_mha kernels (prefix)");
    a.p_items = 0;
    launch_items(a, z, 0, p.o_tile, (unsigned)o_items, ctx->stream);
  } else {
    a.p_items = (int)p_items;
    launch_items(a, z, p.pooled ? p.p_tile : 0, p.o_tile, (unsigned)(p_items + o_items), ctx->stream);
  }
  AUR_LAUNCH_CHECK(ctx, "paged_mha kernels");
  if (floats) {
    int lanes = 2;  // of a row: a power of two of them, 4 columns each
    while (4 * lanes < a.dh) lanes *= 2;
    const int turns = (p.parts() * lanes + 63) / 64;
    auto* join = turns <= 1 ? paged_join_kernel<1> : turns <= 2 ? paged_join_kernel<2>
                 : turns <= 4 ? paged_join_kernel<4> : paged_join_kernel<8>;
    hipLaunchKernelGGL(join, dim3((unsigned)rows4), dim3(256), 0, ctx->stream, a, lanes);
    AUR_LAUNCH_CHECK(ctx, "paged_join_kernel");
  }
  return 0;
}

}  // extern "C"
