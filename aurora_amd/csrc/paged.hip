// Appending to a paged K/V cache with the position rotation on the way, and
// the cos / sin table that it reads.
//
// New token i of a sequence with n new tokens and L own ones (the new ones
// among them) has the own index j = L - n + i and stands at position P + j
// behind the shared prefix of P tokens.  With (c, s) = (cos, sin)(position ·
// θ^(-2u / rot)) a pair (x, y) becomes (x·c − y·s, y·c + x·s); pair u of a head
// is its columns (u, u + rot/2), or (2u, 2u + 1).  Columns from rot on, and V,
// are copied.  Row j of a sequence lies in page pages[s][j / page_len].
//
// One thread moves 4 columns (8 of a rotated pair of halves) of one head of one
// token, whole blocks work on one token, so that its sequence is found once (a
// block-wide count over the offsets, one round trip, where a binary search would
// take log2 b of them).  Bound by HBM for prompts and by the launch for a step:
// 16 prompts of 1024 tokens each, 16 heads of 64: fp32 89 µs, 4.5 TB/s of the 4.9 of a
// large copy, bf16 82 µs, 4.1 TB/s; a step of 32 sequences 5.4 µs, 3.4 of them the
// kernel's.
#include "common.hpp"
#include "paged.hpp"

using namespace aurpaged;

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

struct AppendArgs {
  Batch b;
  const float *q, *k, *v;
  float* q_out;
  void *kp, *vp;
  const float* table;  // [n_pos][rot/2] of (cos, sin)
  int ld_q, ld_kv, ld_qo;
  int H, Hkv, dh, rot, n_pages, sh;
  bool pairs;
};

// Rounded to the nearest bf16, ties to even.
__device__ __forceinline__ void put(float* p, floatx4 x) { *reinterpret_cast<floatx4*>(p) = x; }
__device__ __forceinline__ void put(__bf16* p, floatx4 x) {
  *reinterpret_cast<bf16x4*>(p) = __builtin_convertvector(x, bf16x4);
}

template <class T>
__device__ __forceinline__ void move(const AppendArgs& a, const float* src, T* dst, int u, const float* tab,
                                     bool rotate) {
  const int half = a.rot / 2;
  auto get = [&](int c) { return *reinterpret_cast<const floatx4*>(src + c); };
  if (!rotate || 4 * u >= (a.pairs ? a.rot : half)) {  // copied columns, after the rotated ones
    const int c = 4 * u + (rotate && !a.pairs ? half : 0);
    put(dst + c, get(c));
    return;
  }
  const floatx4 t0 = *reinterpret_cast<const floatx4*>(tab + (a.pairs ? 4 : 8) * u);
  const floatx4 x = get(4 * u);
  if (a.pairs) {
    put(dst + 4 * u, floatx4{x[0] * t0[0] - x[1] * t0[1], x[1] * t0[0] + x[0] * t0[1],
                             x[2] * t0[2] - x[3] * t0[3], x[3] * t0[2] + x[2] * t0[3]});
    return;
  }
  const floatx4 t1 = *reinterpret_cast<const floatx4*>(tab + 8 * u + 4);
  const floatx4 y = get(4 * u + half);
  const floatx4 c = {t0[0], t0[2], t1[0], t1[2]}, s = {t0[1], t0[3], t1[1], t1[3]};
  put(dst + 4 * u, x * c - y * s);
  put(dst + 4 * u + half, y * c + x * s);
}

template <class T>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a, int blocks_per_token) {
  const int t = blockIdx.x / blocks_per_token;
  const int s = sequence_of(a.b, t);
  if (s >= a.b.b) return;  // a row behind the last sequence
  const Seq q = sequence(a.b, s);
  const int i = t - q.lo;
  if (i < 0 || i >= q.n) return;
  const int j = q.len - q.n + i;
  if (j < 0) return;  // fewer own tokens than new ones: this one has no place
  const float* tab = a.table + (size_t)(a.b.prefix_len + j) * a.rot;
  const int per_rot = a.dh / 4 - (a.pairs ? 0 : a.rot / 8);  // units of a rotated head
  int u = (blockIdx.x % blocks_per_token) * 256 + threadIdx.x;
  if (u < a.H * per_rot) {
    if (a.q_out) {
      const int h = u / per_rot;
      move(a, a.q + (size_t)t * a.ld_q + h * a.dh, a.q_out + (size_t)t * a.ld_qo + h * a.dh, u - h * per_rot, tab,
           a.rot > 0);
    }
    return;
  }
  u -= a.H * per_rot;
  const int page = a.b.pages[(size_t)s * a.b.max_pages + (j >> a.sh)];
  if ((unsigned)page >= (unsigned)a.n_pages) return;  // no page there: the row is dropped
  const size_t row = ((size_t)page << a.sh) + (j & ((1 << a.sh) - 1));
  const bool is_k = u < a.Hkv * per_rot;
  if (!is_k) u -= a.Hkv * per_rot;
  const int per = is_k ? per_rot : a.dh / 4;
  const int h = u / per;
  if (h >= a.Hkv) return;
  const size_t dst = (row * a.Hkv + h) * a.dh;
  move(a, (is_k ? a.k : a.v) + (size_t)t * a.ld_kv + h * a.dh, static_cast<T*>(is_k ? a.kp : a.vp) + dst, u - h * per,
       tab, is_k && a.rot > 0);
}

// Angles in 64 bits: at position 10^6 a 32-bit product of position and frequency is off by
// up to 2^-5, and so would its cos and sin be.
__global__ void __launch_bounds__(256) rotary_table_kernel(float* table, double log2_theta, int half, long long n) {
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  const int u = (int)(e % half);
  const double pos = (double)(e / half);
  double s, c;
  sincos(pos * exp2(-log2_theta * u / half), &s, &c);
  table[2 * e] = (float)c;
  table[2 * e + 1] = (float)s;
}

}  // namespace

namespace aurpaged {

int check_paged(aur_ctx* ctx, const char* who, const aur_paged_cache* c, const aur_paged_batch* b, Batch* out) {
  using aur::set_error;
  if (!c || !b) return set_error(ctx, AUR_EINVAL, "%s: null cache or batch", who);
  if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v))
    return set_error(ctx, AUR_EINVAL, "%s: the pools must be there and 16-byte aligned", who);
  if (c->dtype != AUR_PAGED_F32 && c->dtype != AUR_PAGED_BF16)
    return set_error(ctx, AUR_EINVAL, "%s: dtype %u", who, c->dtype);
  if (c->n_pages == 0 || c->page_len == 0 || (c->page_len & (c->page_len - 1)) || c->n_kv_head == 0 || c->d_head == 0)
    return set_error(ctx, AUR_EINVAL, "%s: n_pages=%u page_len=%u (a power of two) n_kv_head=%u d_head=%u", who,
                     c->n_pages, c->page_len, c->n_kv_head, c->d_head);
  if (c->d_head % 8 != 0 || c->d_head > 128)
    return set_error(ctx, AUR_ELIMIT, "%s: d_head=%u (multiples of 8 up to 128)", who, c->d_head);
  if ((uint64_t)c->n_pages * c->page_len > 0x7fffffffu || c->n_kv_head > 4096)
    return set_error(ctx, AUR_ELIMIT, "%s: pool of %u pages of %u rows, n_kv_head=%u", who, c->n_pages, c->page_len,
                     c->n_kv_head);
  if (b->n_tok > 0x00ffffffu || b->b > 0x00ffffffu)
    return set_error(ctx, AUR_ELIMIT, "%s: n_tok=%u b=%u", who, b->n_tok, b->b);
  if (b->b && b->n_tok) {
    if (!b->tok_off || !b->own_len || (b->max_own && !b->pages) || (b->prefix_len && !b->prefix_pages))
      return set_error(ctx, AUR_EINVAL, "%s: null array in the batch", who);
    if (b->max_tok == 0) return set_error(ctx, AUR_EINVAL, "%s: max_tok=0", who);
  }
  if (b->max_own > (uint64_t)b->max_pages * c->page_len)
    return set_error(ctx, AUR_EINVAL, "%s: max_own=%u in %u pages of %u", who, b->max_own, b->max_pages, c->page_len);
  if (b->prefix_len > (uint64_t)b->n_prefix_pages * c->page_len)
    return set_error(ctx, AUR_EINVAL, "%s: prefix_len=%u in %u pages of %u", who, b->prefix_len, b->n_prefix_pages,
                     c->page_len);
  // positions stay below 2^30, so that a tile's end past the last key is an int too
  if ((uint64_t)b->prefix_len + b->max_own > 0x3fffffffu || b->max_pages > 0x3fffffffu)
    return set_error(ctx, AUR_ELIMIT, "%s: prefix_len=%u + max_own=%u", who, b->prefix_len, b->max_own);
  *out = Batch{b->tok_off,     b->own_len, b->pages, b->prefix_pages, (int)b->b, (int)b->max_pages, (int)b->n_tok,
               (int)(b->max_tok < b->n_tok ? b->max_tok : b->n_tok), (int)b->max_own, (int)b->prefix_len};
  return 0;
}

}  // namespace aurpaged

extern "C" {

int aur_rotary_table(aur_ctx* ctx, float* table, uint32_t n_pos, uint32_t rot_dim, float theta) {
  AUR_CHECK_CTX(ctx);
  if (!table || n_pos == 0 || rot_dim == 0 || rot_dim % 2 || !(theta > 0.f) || theta > 3.4e38f)
    return aur::set_error(ctx, AUR_EINVAL, "aur_rotary_table: n_pos=%u rot_dim=%u (even) theta=%g", n_pos, rot_dim,
                          (double)theta);
  const long long n = (long long)n_pos * (rot_dim / 2), blocks = (n + 255) / 256;
  if (blocks > kMaxBlocks) return aur::set_error(ctx, AUR_ELIMIT, "aur_rotary_table: n_pos=%u rot_dim=%u", n_pos, rot_dim);
  hipLaunchKernelGGL(rotary_table_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, table,
                     log2((double)theta), (int)(rot_dim / 2), n);
  AUR_LAUNCH_CHECK(ctx, "rotary_table_kernel");
  return 0;
}

int aur_kv_append_paged(aur_ctx* ctx, const aur_paged_cache* cache, const aur_paged_batch* batch, const float* q,
                        uint32_t ld_q, const float* k, const float* v, uint32_t ld_kv, float* q_out, uint32_t ld_qo,
                        const float* table, uint32_t n_pos, uint32_t rot_dim, uint32_t n_head, int pairs) {
  AUR_CHECK_CTX(ctx);
  const char* who = "aur_kv_append_paged";
  AppendArgs a{};
  if (int rc = check_paged(ctx, who, cache, batch, &a.b)) return rc;
  const uint32_t dh = cache->d_head, row = cache->n_kv_head * dh;
  if (rot_dim > dh || rot_dim % 8 != 0)
    return aur::set_error(ctx, AUR_EINVAL, "%s: rot_dim=%u of d_head=%u (a multiple of 8)", who, rot_dim, dh);
  if (rot_dim && (!table || !aligned16(table) || (uint64_t)a.b.prefix_len + a.b.max_own > n_pos))
    return aur::set_error(ctx, AUR_EINVAL, "%s: table of %u positions (16-byte aligned), %d + %d needed", who, n_pos,
                          a.b.prefix_len, a.b.max_own);
  if ((q == nullptr) != (q_out == nullptr))
    return aur::set_error(ctx, AUR_EINVAL, "%s: q and q_out come together", who);
  if (q && (n_head == 0 || n_head % cache->n_kv_head != 0))
    return aur::set_error(ctx, AUR_EINVAL, "%s: n_head=%u, a multiple of n_kv_head=%u", who, n_head, cache->n_kv_head);
  if (n_head > 4096) return aur::set_error(ctx, AUR_ELIMIT, "%s: n_head=%u", who, n_head);
  if (a.b.b == 0 || a.b.n_tok == 0) return 0;
  if (!k || !v || !aligned16(k) || !aligned16(v) || !aligned16(q) || !aligned16(q_out))
    return aur::set_error(ctx, AUR_EINVAL, "%s: k and v must be there, all rows 16-byte aligned", who);
  const uint32_t qd = q ? n_head * dh : 0;
  if (ld_kv < row || ld_kv % 4 || ld_kv > 0x7fffffffu || (q && (ld_q < qd || ld_qo < qd || ld_q % 4 || ld_qo % 4 ||
                                                               ld_q > 0x7fffffffu || ld_qo > 0x7fffffffu)))
    return aur::set_error(ctx, AUR_EINVAL, "%s: ld_q=%u ld_kv=%u ld_qo=%u (multiples of 4, at least a row)", who, ld_q,
                          ld_kv, ld_qo);
  if (q && q == q_out && ld_q != ld_qo && a.b.n_tok > 1)  // a row's result would lie on another's input
    return aur::set_error(ctx, AUR_EINVAL, "%s: q and q_out one buffer with ld_q=%u, ld_qo=%u", who, ld_q, ld_qo);
  a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.kp = cache->k; a.vp = cache->v; a.table = table;
  a.ld_q = (int)ld_q; a.ld_kv = (int)ld_kv; a.ld_qo = (int)ld_qo;
  a.H = q ? (int)n_head : 0; a.Hkv = (int)cache->n_kv_head; a.dh = (int)dh; a.rot = (int)rot_dim;
  a.n_pages = (int)cache->n_pages; a.sh = log2_of(cache->page_len); a.pairs = pairs != 0;
  const int per_rot = a.dh / 4 - (a.pairs ? 0 : a.rot / 8);
  const int units = (a.H + a.Hkv) * per_rot + a.Hkv * a.dh / 4;
  const int per_token = (units + 255) / 256;
  const uint64_t blocks = (uint64_t)a.b.n_tok * per_token;
  if (blocks > kMaxBlocks) return aur::set_error(ctx, AUR_ELIMIT, "%s: n_tok=%d rows of %d heads", who, a.b.n_tok, a.H);
  if (cache->dtype == AUR_PAGED_F32)
    hipLaunchKernelGGL(append_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, a, per_token);
  else
    hipLaunchKernelGGL(append_kernel<__bf16>, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, a, per_token);
  AUR_LAUNCH_CHECK(ctx, "append_kernel");
  return 0;
}

}  // extern "C"
