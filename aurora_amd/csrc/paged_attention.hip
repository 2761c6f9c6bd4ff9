// Attention of new tokens over a paged K/V cache, for sequences that share a
// prefix.  Query row (token (s, i), head h) sees the P keys of the prefix and
// its sequence's own keys 0 .. j, j = L − n + i:
//   out = Σ softmax(q·k / √d_head) v,   lse = log Σ exp(q·k / √d_head);
// a row that sees no key gets out 0, lse −∞.
//
// Work is cut into items (one block each): up to 16·RT query rows that read the
// same keys, and a range of those keys.
//   * Pooled (few rows a sequence, as in decode): the rows of ALL sequences of one
//     K/V head against a range of the prefix, so the prefix is read once for all,
//     and the rows of one sequence against a range of its own keys.
//   * Otherwise the rows of one sequence against prefix and own keys as one axis.
// Where a row's keys are cut into several ranges, items leave (m, l, Σ p v) and a
// second launch joins them in the order of the ranges: the result does not
// depend on which block ends first.
//
// In an item each of the block's 4 waves takes every fourth group of 32 keys and
// keeps its own running maximum and sum; the waves are joined through LDS in
// their order.  K and V go from the pools straight into the registers that feed
// the MFMA, both as 16-byte loads: Sᵀ = K·Qᵀ takes 4 consecutive columns of a key
// per lane (the four MFMAs that they feed use them as k = 0 … 3 of 4 lane groups),
// its result is, as it lies, the B operand of Oᵀ += Vᵀ·Pᵀ, and there a lane's 4
// consecutive columns of V are rows of four MFMAs (row r of MFMA c is column
// 4r + c), so V needs no transposition.
#include "attention.hpp"
#include "common.hpp"
#include "paged.hpp"

using namespace aurattn;
using namespace aurpaged;

namespace {

constexpr int NW = 4;         // waves of a block
constexpr int STEP = 32;      // keys of a wave's step
constexpr float LN2 = 0.6931471805599453f;

struct MhaArgs {
  Batch b;
  const float* q;
  float *out, *lse;
  const void *k, *v;
  float *part_o, *part_ml;  // [part][token][H][dh], [part][token][H][2]; null: items write out and lse
  int ld_q, ld_o;
  int H, Hkv, G, dh, n_pages, sh;
  float scale;
  // The plan: row tiles and key ranges of the prefix's items and the own ones.
  int pooled;
  int p_tiles, p_splits, p_keys;  // p_keys keys a range
  int o_tiles, o_splits, o_keys;
  int p_items;                    // items 0 .. p_items-1 are the prefix's
};

__device__ __forceinline__ floatx4 load4(const float* p) { return *reinterpret_cast<const floatx4*>(p); }
__device__ __forceinline__ floatx4 load4(const __bf16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return floatx4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                 __uint_as_float(u.y & 0xffff0000u)};
}

// DT: d_head in blocks of 16 columns, rounded up.
template <class T, int DT, int RT>
__global__ void __launch_bounds__(64 * NW) paged_mha_kernel(MhaArgs a) {
  constexpr int VB = (DT + 3) / 4;  // blocks of 64 columns of V
  constexpr int KT = STEP / 16;
  constexpr int R = 16 * RT, OS = 64 * VB + 4;
  __shared__ float sm[NW][R], sl[NW][R];
  __shared__ __attribute__((aligned(16))) float so[R][OS];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int g = lane >> 4, l16 = lane & 15;
  const float sl2 = a.scale * LOG2E;

  // Which rows, which keys.  Key x < pre of the item's axis is the prefix's x, others are own.
  int item = blockIdx.x, s = 0, part, x0, x1, row0, n_rows, tok0, pre, first = 0;
  const bool of_prefix = item < a.p_items;
  int hk;
  if (of_prefix) {
    hk = item % a.Hkv;
    item /= a.Hkv;
    const int tile = item % a.p_tiles;
    part = item / a.p_tiles;
    tok0 = 0;
    row0 = tile * R;
    n_rows = a.b.n_tok * a.G;
    pre = a.b.prefix_len;
    x0 = part * a.p_keys;
    x1 = min(x0 + a.p_keys, pre);
  } else {
    item -= a.p_items;
    hk = item % a.Hkv;
    item /= a.Hkv;
    const int tile = item % a.o_tiles;
    item /= a.o_tiles;
    s = item % a.b.b;
    part = item / a.b.b;
    const Seq q = sequence(a.b, s);
    tok0 = q.lo;
    row0 = tile * R;
    n_rows = q.n * a.G;
    pre = a.pooled ? 0 : a.b.prefix_len;
    x0 = part * a.o_keys;
    if (row0 >= n_rows || (part > 0 && x0 >= pre + q.len)) return;
    first = pre + q.len - q.n + 1;  // keys that the sequence's first new token sees
    x1 = min(x0 + a.o_keys, max(first + (min(row0 + R, n_rows) - 1) / a.G, pre));
    if (a.pooled) part += a.p_splits;
  }

  // Rows of this lane (one per tile of 16): token, head and how many keys of the axis it sees.
  int vis[RT];
  floatx4 qf[RT][DT];
  int vmin = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = row0 + 16 * r + l16;
    const bool live = row < n_rows;
    const int t = live ? row / a.G : 0, h = hk * a.G + (live ? row - t * a.G : 0);
    vis[r] = !live ? 0 : of_prefix ? pre : max(first + t, pre);
    if (live) vmin = min(vmin, vis[r]);
    const float* qp = a.q + (size_t)(tok0 + t) * a.ld_q + (size_t)h * a.dh;
#pragma unroll
    for (int c = 0; c < DT; ++c) {
      const int col = 16 * c + 4 * g;
      qf[r][c] = live && col < a.dh ? load4(qp + col) * sl2 : floatx4{0.f, 0.f, 0.f, 0.f};
    }
  }
#pragma unroll
  for (int m = 1; m < 16; m *= 2) vmin = min(vmin, __shfl_xor(vmin, m, 64));

  const T* kp = static_cast<const T*>(a.k);
  const T* vp = static_cast<const T*>(a.v);
  const size_t ld = (size_t)a.Hkv * a.dh;
  const size_t head = (size_t)hk * a.dh;
  // Pool row of key x, or −1 where there is none.
  auto place = [&](int x) {
    if (x >= x1) return -1;
    const bool p = x < pre;
    const int i = p ? x : x - pre;
    const int page = p ? a.b.prefix_pages[i >> a.sh] : a.b.pages[(size_t)s * a.b.max_pages + (i >> a.sh)];
    return (unsigned)page < (unsigned)a.n_pages ? (page << a.sh) + (i & ((1 << a.sh) - 1)) : -1;
  };
  floatx4 kf[KT][DT], vf[KT][4][VB];
  auto load_k = [&](int at) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const T* p = kp + (size_t)max(__shfl(at, 16 * kt + l16, 64), 0) * ld + head;
#pragma unroll
      for (int c = 0; c < DT; ++c) {
        const int col = 16 * c + 4 * g;
        kf[kt][c] = DT * 16 == a.dh || col < a.dh ? load4(p + col) : floatx4{0.f, 0.f, 0.f, 0.f};
      }
    }
  };
  auto load_v = [&](int at) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = __shfl(at, 16 * kt + 4 * g + e, 64);
        const T* p = vp + (size_t)max(row, 0) * ld + head;
#pragma unroll
        for (int b = 0; b < VB; ++b) {
          const int col = 64 * b + 4 * l16;
          // a key that is not there adds nothing, whatever lies in the row
          vf[kt][e][b] = row >= 0 && col < a.dh ? load4(p + col) : floatx4{0.f, 0.f, 0.f, 0.f};
        }
      }
  };

  floatx4 acc[RT][VB][4];
  float m[RT], l[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[r][b][c] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  int x = x0 + STEP * w;
  int at = place(x + (lane & 31));
  if (x < x1) load_k(at);
  for (; x < x1; x += STEP * NW) {
    load_v(at);
    const unsigned long long there = __ballot(at >= 0);
    const int at_next = place(x + STEP * NW + (lane & 31));
    floatx4 st[RT][KT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        st[r][kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) st[r][kt] = mfma16x16x4(kf[kt][c][e], qf[r][c][e], st[r][kt]);
      }
    if (x + STEP * NW < x1) load_k(at_next);
    at = at_next;
    const bool mixed = x + STEP > vmin;  // some row does not see some key
    bool odd = false;                    // … and a value that 0 times would not remove is there
    if (mixed) {
      float z = 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int b = 0; b < VB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) z += 0.f * vf[kt][e][b][i];
      odd = __ballot(!(z == 0.f)) != 0;
    }
    const bool masked = mixed || there != ~0ull;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (masked) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = 16 * kt + 4 * g + e;
            if (x + key >= vis[r] || !(there >> key & 1)) st[r][kt][e] = -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        mx = fmaxf(mx, fmaxf(fmaxf(st[r][kt][0], st[r][kt][1]), fmaxf(st[r][kt][2], st[r][kt][3])));
      const float m_new = fmaxf(m[r], rows4_max(mx));
      const float ms = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m[r] - ms);
      m[r] = m_new;
      float ps = 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          st[r][kt][e] = __builtin_amdgcn_exp2f(st[r][kt][e] - ms);
          ps += st[r][kt][e];
        }
      l[r] = l[r] * alpha + ps;
#pragma unroll
      for (int b = 0; b < VB; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][b][c] *= alpha;
    }
    if (!odd) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int b = 0; b < VB; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int r = 0; r < RT; ++r)
                acc[r][b][c] = mfma16x16x4(vf[kt][e][b][c], st[r][kt][e], acc[r][b][c]);
    } else {
      // An infinity or NaN among values that not every row sees: each row adds only those it does.
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll 1
            for (int kg = 0; kg < 4; ++kg) {
              const float p = __shfl(st[r][kt][e], 16 * kg + l16, 64);
              const int key = 16 * kt + 4 * kg + e;
              const bool seen = x + key < vis[r] && (there >> key & 1);
#pragma unroll
              for (int b = 0; b < VB; ++b)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const float v = __shfl(vf[kt][e][b][c], 16 * kg + 4 * g + i, 64);
                    if (seen) acc[r][b][c][i] += p * v;
                  }
            }
    }
  }

  // Join the four waves: common maximum, then their sums added in wave order.
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] = rows4_sum(l[r]);
    if (g == 0) {
      sm[w][16 * r + l16] = m[r];
      sl[w][16 * r + l16] = l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < NW; ++i) M = fmaxf(M, sm[i][16 * r + l16]);
    const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - M);
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[r][b][c] *= f;
  }
  for (int i = 0; i < NW; ++i) {
    if (w == i) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int b = 0; b < VB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            floatx4* p = reinterpret_cast<floatx4*>(&so[16 * r + l16][64 * b + 16 * g + 4 * j]);
            const floatx4 v = {acc[r][b][0][j], acc[r][b][1][j], acc[r][b][2][j], acc[r][b][3][j]};
            *p = i == 0 ? v : *p + v;
          }
    }
    __syncthreads();
  }
  const int n4 = a.dh / 4;
  for (int i = tid; i < R * n4; i += 64 * NW) {
    const int r = i / n4, c = 4 * (i - r * n4), row = row0 + r;
    if (row >= n_rows) break;
    const int t = row / a.G, h = hk * a.G + row - t * a.G;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int j = 0; j < NW; ++j) M = fmaxf(M, sm[j][r]);
#pragma unroll
    for (int j = 0; j < NW; ++j) L += (M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sm[j][r] - M)) * sl[j][r];
    const floatx4 o = *reinterpret_cast<const floatx4*>(&so[r][c]);
    const size_t token = (size_t)tok0 + t;
    if (a.part_o) {
      const size_t rec = ((size_t)part * a.b.n_tok + token) * a.H + h;
      *reinterpret_cast<floatx4*>(a.part_o + rec * a.dh + c) = o;
      if (c == 0) {
        a.part_ml[2 * rec] = M;
        a.part_ml[2 * rec + 1] = L;
      }
    } else {
      *reinterpret_cast<floatx4*>(a.out + token * a.ld_o + (size_t)h * a.dh + c) = L == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : o * (1.f / L);
      if (c == 0 && a.lse) a.lse[token * a.H + h] = L == 0.f ? -INFINITY : (M + __log2f(L)) * LN2;
    }
  }
}

// out and lse of a token's rows from the records of their ranges, in the ranges' order.
__global__ void __launch_bounds__(256) paged_join_kernel(MhaArgs a) {
  const int t = blockIdx.x;
  const int s = sequence_of(a.b, t);
  if (s >= a.b.b) return;  // a row behind the last sequence
  const Seq q = sequence(a.b, s);
  if (t < q.lo || t - q.lo >= q.n) return;
  const int axis = q.len + (a.pooled ? 0 : a.b.prefix_len);
  const int np = a.p_splits + max((axis + a.o_keys - 1) / a.o_keys, 1);  // range 0 is always written
  const int n4 = a.dh / 4;
  const size_t step = (size_t)a.b.n_tok * a.H;
  for (int i = threadIdx.x; i < a.H * n4; i += 256) {
    const int h = i / n4, c = 4 * (i - h * n4);
    size_t rec = (size_t)t * a.H + h;
    float M = -INFINITY, L = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < np; ++p, rec += step) {
      const float m = a.part_ml[2 * rec], l = a.part_ml[2 * rec + 1];
      const floatx4 v = load4(a.part_o + rec * a.dh + c);
      const float M1 = fmaxf(M, m), ms = M1 == -INFINITY ? 0.f : M1;
      // a record without a maximum was summed against 0
      const float f = M == -INFINITY ? (M1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(-ms)) : __builtin_amdgcn_exp2f(M - ms);
      const float e = m == -INFINITY ? (M1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(-ms)) : __builtin_amdgcn_exp2f(m - ms);
      L = L * f + l * e;
      o = o * f + v * e;
      M = M1;
    }
    *reinterpret_cast<floatx4*>(a.out + (size_t)t * a.ld_o + (size_t)h * a.dh + c) =
        L == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : o * (1.f / L);
    if (c == 0 && a.lse) a.lse[(size_t)t * a.H + h] = L == 0.f ? -INFINITY : (M + __log2f(L)) * LN2;
  }
}

// How a call is cut into items, from what the host knows; the scratch's size follows from it.
struct Plan {
  int pooled, p_rt, o_rt, p_tiles, p_splits, p_keys, o_tiles, o_splits, o_keys;
  int parts() const { return p_splits + o_splits; }
};

int tiles_of(long long rows, int* rt) {
  *rt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  return (int)((rows + 16 * *rt - 1) / (16 * *rt));
}

constexpr uint32_t kMaxRows = 0x7fffff00u;  // query rows of a call, and a tile more, are ints
constexpr int kItems = 1024;  // blocks that a launch aims at: 4 of each CU

Plan make_plan(const Batch& b, int Hkv, int G) {
  Plan p{};
  const int P = b.prefix_len;
  p.pooled = P > 0 && b.b > 1 && (long long)b.max_tok * G < 64;
  p.o_tiles = tiles_of((long long)b.max_tok * G, &p.o_rt);
  p.p_rt = 1;
  if (p.pooled) p.p_tiles = tiles_of((long long)b.n_tok * G, &p.p_rt);
  const int axis = b.max_own + (p.pooled ? 0 : P);
  const int block = STEP * NW;
  const double work = (double)Hkv * ((double)p.p_tiles * P + (double)b.b * p.o_tiles * axis);
  const double want = work / kItems;
  int keys = want > 1e9 ? 1000000000 : ((int)want + block - 1) / block * block;
  if (keys < block) keys = block;
  p.p_keys = p.o_keys = keys;
  p.p_splits = p.pooled ? (P + keys - 1) / keys : 0;
  p.o_splits = axis > keys ? (axis + keys - 1) / keys : 1;
  return p;
}

size_t ws_floats(const Plan& p, const Batch& b, int H, int dh) {
  return p.parts() > 1 ? (size_t)p.parts() * b.n_tok * H * (dh + 2) : 0;
}

template <class T, int DT>
void launch_rt(const MhaArgs& a, int rt, unsigned items, hipStream_t st) {
  const dim3 g(items), b(64 * NW);
  if (rt == 1)
    hipLaunchKernelGGL((paged_mha_kernel<T, DT, 1>), g, b, 0, st, a);
  else if (rt == 2)
    hipLaunchKernelGGL((paged_mha_kernel<T, DT, 2>), g, b, 0, st, a);
  else
    hipLaunchKernelGGL((paged_mha_kernel<T, DT, 4>), g, b, 0, st, a);
}

template <class T>
void launch_dt(const MhaArgs& a, int rt, unsigned items, hipStream_t st) {
  const int dt = (a.dh + 15) / 16;
  if (dt == 1) launch_rt<T, 1>(a, rt, items, st);
  else if (dt == 2) launch_rt<T, 2>(a, rt, items, st);
  else if (dt == 3) launch_rt<T, 3>(a, rt, items, st);
  else if (dt == 4) launch_rt<T, 4>(a, rt, items, st);
  else if (dt <= 6) launch_rt<T, 6>(a, rt, items, st);
  else launch_rt<T, 8>(a, rt, items, st);
}

void launch_items(const MhaArgs& a, bool f32, int rt, unsigned items, hipStream_t st) {
  f32 ? launch_dt<float>(a, rt, items, st) : launch_dt<__bf16>(a, rt, items, st);
}

}  // namespace

extern "C" {

size_t aur_mha_paged_ws_bytes(const aur_paged_cache* cache, const aur_paged_batch* batch, uint32_t n_head) {
  Batch b;
  if (check_paged(nullptr, "aur_mha_paged_ws_bytes", cache, batch, &b) != 0 || n_head == 0 || n_head > 4096 ||
      (uint64_t)b.n_tok * n_head > kMaxRows || n_head % cache->n_kv_head != 0 || b.b == 0 || b.n_tok == 0)
    return 0;
  return 4 * ws_floats(make_plan(b, (int)cache->n_kv_head, (int)(n_head / cache->n_kv_head)), b, (int)n_head,
                       (int)cache->d_head);
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
  const Plan p = make_plan(a.b, a.Hkv, a.G);
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
  const uint64_t p_items = (uint64_t)a.Hkv * p.p_tiles * p.p_splits;
  const uint64_t o_items = (uint64_t)a.Hkv * p.o_tiles * a.b.b * p.o_splits;
  if (p_items > kMaxBlocks || o_items > kMaxBlocks)
    return aur::set_error(ctx, AUR_ELIMIT, "%s: %llu + %llu blocks", who, (unsigned long long)p_items,
                          (unsigned long long)o_items);
  const bool f32 = cache->dtype == AUR_PAGED_F32;
  if (p.pooled) {
    a.p_items = (int)p_items;
    launch_items(a, f32, p.p_rt, (unsigned)p_items, ctx->stream);
    AUR_LAUNCH_CHECK(ctx, "paged_mha_kernel (prefix)");
    a.p_items = 0;
  }
  launch_items(a, f32, p.o_rt, (unsigned)o_items, ctx->stream);
  AUR_LAUNCH_CHECK(ctx, "paged_mha_kernel");
  if (floats) {
    hipLaunchKernelGGL(paged_join_kernel, dim3(a.b.n_tok), dim3(256), 0, ctx->stream, a);
    AUR_LAUNCH_CHECK(ctx, "paged_join_kernel");
  }
  return 0;
}

}  // extern "C"
