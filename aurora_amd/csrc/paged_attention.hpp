// Attention of new tokens over a paged K/V cache, for sequences that share a
// prefix.  Query row (token (s, i), head h) sees the P keys of the prefix and
// its sequence's own keys 0 .. j, j = L − n + i:
//   out = Σ softmax(q·k / √d_head) v,   lse = log Σ exp(q·k / √d_head);
// a row that sees no key gets out 0, lse −∞.  Scores carry log2(e) from the
// queries on, so that every exponential is an exp2.
//
// Work is cut into items (one block each): query rows that read the same keys,
// and a range of those keys.
//   * Pooled (few rows a sequence, as in decode): the rows of ALL sequences of one
//     K/V head against a range of the prefix, so the prefix is read once for all,
//     and the rows of one sequence against a range of its own keys.
//   * Otherwise the rows of one sequence against prefix and own keys as one axis.
// Where a row's keys are cut into several ranges, items leave (m, l, Σ p v) in the
// caller's scratch and a second launch joins them in the order of the ranges: the
// result does not depend on which block ends first.
//
// Three kinds of items, by their rows:
//   few_item   one token, 1 to 4 rows: vector instructions, bound by reading the keys
//   rows_item  up to 16 rows: keys from the pools straight into the registers that
//              feed the MFMA, bound by reading them and by the MFMA's cycles
//   tile_item  64, 128 or 256 rows: keys laid down in LDS, bound by the MFMA
#pragma once

#include "attention.hpp"
#include "attention_split.hpp"
#include "common.hpp"
#include "lanes.hpp"
#include "paged.hpp"
#include "paged_plan.hpp"

#include <cmath>
#include <type_traits>

using namespace aurattn;
using namespace aurpaged;

namespace aurpaged {

struct MhaArgs {
  Batch b;
  const float* q;
  float *out, *lse;
  const void *k, *v;
  float *part_o, *part_ml;  // [part][token][H][dh], [part][token][H][2]; null: items write out and lse
  int ld_q, ld_o;
  int H, Hkv, G, dh, n_pages, sh;
  const uint8_t *k_scale, *v_scale;  // of e4m3 pools
  int ssh;
  float scale;
  // The plan: row tiles and key ranges of the prefix's items and the own ones.
  int pooled;
  int p_tiles, p_splits, p_keys;  // p_keys keys a range
  int o_tiles, o_splits, o_keys;
  int p_items;                    // items 0 .. p_items-1 are the prefix's
  bool by_xcd;                    // the K/V heads of the same keys run on the same XCD
};

// The dice take blocks in turn, and each has an L2 of its own with lines of 128 bytes.  Where a head's row is
// shorter than that, the items of all K/V heads on the same keys go to one die, one after the other, so that a
// line is fetched once and not by every die that wants a part of it (64 sequences of 512 to 1024 keys, 16 heads of 64
// in e4m3, out of the chip's caches: 40 us without this order, 24 with it).  With fewer than kDice sets of such items
// some dice would have none.
constexpr int kDice = 8;
inline bool heads_by_xcd(int row_bytes, uint64_t p_groups, uint64_t o_groups) {
  return row_bytes < 128 && o_groups >= kDice && (p_groups == 0 || p_groups >= kDice);
}
// Blocks for `groups` sets of items, a K/V head each.
inline uint64_t items_of(bool by_xcd, uint64_t groups, int n_kv_head) {
  return (by_xcd ? (groups + kDice - 1) / kDice * kDice : groups) * n_kv_head;
}

// Launches a call's items for pools of each type: own items of z's rows where the tile is 16, prefix items of
// p_tile beside them (0: items of one kind).
void launch_items_f32(const MhaArgs& a, const Sizes& z, int p_tile, int tile, unsigned items, hipStream_t st);
void launch_items_bf16(const MhaArgs& a, const Sizes& z, int p_tile, int tile, unsigned items, hipStream_t st);
void launch_items_e4m3(const MhaArgs& a, const Sizes& z, int p_tile, int tile, unsigned items, hipStream_t st);

}  // namespace aurpaged

namespace {

constexpr int NW = 4;         // waves of a block
constexpr int STEP = 32;      // keys of a wave's step
constexpr float LN2 = 0.6931471805599453f;

typedef unsigned uint2v __attribute__((ext_vector_type(2)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- an item

struct Item {
  int s, hk, part;
  int row0, n_rows, tok0;  // first query row, how many rows there are, the token of row 0
  int x0, x1;              // keys of the axis
  int pre, first;          // the axis's prefix keys; keys that row 0's token sees
  bool of_prefix;
};

// Key x of the axis is the prefix's while x < pre, then the sequence's own.  The page's number can
// be asked for before the sequence's length is known: the table is read inside its bounds anyway.
__device__ __forceinline__ int page_of(const MhaArgs& a, int s, int pre, int x) {
  if (x < pre) return a.b.prefix_pages[min(x, a.b.prefix_len - 1) >> a.sh];
  return a.b.max_own > 0 ? a.b.pages[(size_t)s * a.b.max_pages + min((x - pre) >> a.sh, a.b.max_pages - 1)] : -1;
}
// Pool row of key x, or −1 where there is none.
__device__ __forceinline__ int row_of(const MhaArgs& a, const Item& it, int x, int page) {
  const int i = x < it.pre ? x : x - it.pre;
  return x < it.x1 && (unsigned)page < (unsigned)a.n_pages ? (page << a.sh) + (i & ((1 << a.sh) - 1)) : -1;
}

// The block's item; `page` is the page of key x0 + lead.  False: nothing to do.  T: by_xcd is looked at for e4m3
// alone (the other types' steps took 3 % longer with a branch on it).
template <class T, int R>
__device__ __forceinline__ bool take_item(const MhaArgs& a, Item& it, int lead, int& page) {
  int item = blockIdx.x;
  it.of_prefix = item < a.p_items;
  it.s = 0;
  it.tok0 = 0;
  it.first = 0;
  if (!it.of_prefix) item -= a.p_items;
  if (sizeof(T) == 1 && a.by_xcd) {
    const int i = item / kDice;
    it.hk = i % a.Hkv;
    item = i / a.Hkv * kDice + item % kDice;
    if (item >= (it.of_prefix ? a.p_tiles * a.p_splits : a.o_tiles * a.b.b * a.o_splits)) return false;
  } else {
    it.hk = item % a.Hkv;
    item /= a.Hkv;
  }
  if (it.of_prefix) {
    it.row0 = item % a.p_tiles * R;
    it.part = item / a.p_tiles;
    it.n_rows = min(max(a.b.tok_off[a.b.b], 0), a.b.n_tok) * a.G;  // rows behind the last sequence are none
    if (it.row0 >= it.n_rows) return false;
    it.pre = a.b.prefix_len;
    it.x0 = it.part * a.p_keys;
    it.x1 = min(it.x0 + a.p_keys, it.pre);
    page = page_of(a, 0, it.pre, it.x0 + lead);
    return true;
  }
  it.row0 = item % a.o_tiles * R;
  item /= a.o_tiles;
  it.s = item % a.b.b;
  it.part = item / a.b.b;
  it.pre = a.pooled ? 0 : a.b.prefix_len;
  it.x0 = it.part * a.o_keys;
  page = page_of(a, it.s, it.pre, it.x0 + lead);
  const Seq q = sequence(a.b, it.s);
  it.tok0 = q.lo;
  it.n_rows = q.n * a.G;
  if (it.row0 >= it.n_rows || (it.part > 0 && it.x0 >= it.pre + q.len)) return false;
  it.first = it.pre + q.len - q.n + 1;
  it.x1 = min(it.x0 + a.o_keys, max(it.first + (min(it.row0 + R, it.n_rows) - 1) / a.G, it.pre));
  if (a.pooled) it.part += a.p_splits;
  return true;
}

// The lane's rows, one of each tile of 16: the query's address, and how many keys of the axis it sees.
template <int RT>
struct Rows {
  const float* q[RT];  // null: no row
  int vis[RT], vmin;   // vmin: the fewest that a row of the item's tile sees
};
template <int RT>
__device__ __forceinline__ void take_rows(const MhaArgs& a, const Item& it, int row0, int l16, Rows<RT>& r) {
  r.vmin = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int row = row0 + 16 * i + l16, t = row / a.G;
    const bool live = row < it.n_rows;
    r.q[i] = live ? a.q + (size_t)(it.tok0 + t) * a.ld_q + (size_t)(it.hk * a.G + row - t * a.G) * a.dh : nullptr;
    r.vis[i] = !live ? 0 : it.of_prefix ? it.pre : max(it.first + t, it.pre);
    if (live) r.vmin = min(r.vmin, r.vis[i]);
  }
#pragma unroll
  for (int m = 1; m < 16; m *= 2) r.vmin = min(r.vmin, __shfl_xor(r.vmin, m, 64));
}

// Running maximum (log2 domain), sum and unnormalised output of RT tiles of 16 rows: lane (g, l16) has row
// l16's m, its own keys' share of l, and in acc[.][b][c][i] the columns 64b + 16g + 4i + c.
template <int DT, int RT>
struct Sums {
  static constexpr int VB = (DT + 3) / 4;
  float m[RT], l[RT];
  floatx4 acc[RT][VB][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int b = 0; b < VB; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][b][c] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
  }
};

// Four columns of a row's result: a record, or the output itself.
__device__ __forceinline__ void store(const MhaArgs& a, const Item& it, int row, int c, floatx4 o, float M, float L) {
  const int t = row / a.G, h = it.hk * a.G + row - t * a.G;
  const size_t token = (size_t)it.tok0 + t;
  if (a.part_o) {
    const size_t rec = ((size_t)it.part * a.b.n_tok + token) * a.H + h;
    *reinterpret_cast<floatx4*>(a.part_o + rec * a.dh + c) = o;
    if (c == 0) {
      a.part_ml[2 * rec] = M;
      a.part_ml[2 * rec + 1] = L;
    }
  } else {
    *reinterpret_cast<floatx4*>(a.out + token * a.ld_o + (size_t)h * a.dh + c) =
        L == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : o * (1.f / L);
    if (c == 0 && a.lse) a.lse[token * a.H + h] = L == 0.f ? -INFINITY : (M + __log2f(L)) * LN2;
  }
}

// ---------------------------------------------------------------- 32 keys in registers

__device__ __forceinline__ floatx4 load4(const float* p) { return *reinterpret_cast<const floatx4*>(p); }

// 32 keys as their loads left them.  K lies as the MFMA takes it (lane (g, l16): key l16 of 16, fp32
// columns 16c + 4g …, bf16 columns 32c + 8g …), of V lane (g, l16) has columns 64b + 4·l16 … of the
// keys 16kt + 4g + e.  `at`: the pool row of key lane % 32, or −1; such a key loads row 0, its score is
// masked and its V taken as zero.  Columns past the head are its last ones again: of K they become
// zeros before use, of V they end in output columns that nobody stores.
template <class T, int DT>
struct Keys32 {
  static constexpr bool F32 = std::is_same<T, float>::value;
  static constexpr int VB = (DT + 3) / 4, KC = F32 ? DT : (DT + 1) / 2;
  using K4 = typename std::conditional<F32, floatx4, uint4v>::type;
  using V4 = typename std::conditional<F32, floatx4, uint2v>::type;
  K4 k[2][KC];
  V4 v[2][4][VB];
  template <bool STREAM>
  __device__ __forceinline__ void load_k(const MhaArgs& a, int hk, int at, int g, int l16) {
    const size_t ld = (size_t)a.Hkv * a.dh;
    const T* kp = static_cast<const T*>(a.k) + (size_t)hk * a.dh;
    constexpr int W = F32 ? 4 : 8;  // columns of a lane's piece
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const T* p = kp + (size_t)max(__shfl(at, 16 * kt + l16, 64), 0) * ld;
#pragma unroll
      for (int c = 0; c < KC; ++c) k[kt][c] = get<STREAM, K4>(p + min(4 * W * c + W * g, a.dh - W));
    }
  }
  template <bool STREAM>
  __device__ __forceinline__ void load_v(const MhaArgs& a, int hk, int at, int g, int l16) {
    const size_t ld = (size_t)a.Hkv * a.dh;
    const T* vp = static_cast<const T*>(a.v) + (size_t)hk * a.dh;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const T* p = vp + (size_t)max(__shfl(at, 16 * kt + 4 * g + e, 64), 0) * ld;
#pragma unroll
        for (int b = 0; b < VB; ++b) v[kt][e][b] = get<STREAM, V4>(p + min(64 * b + 4 * l16, a.dh - 4));
      }
  }
  // STREAM: read once, past the caches.
  template <bool STREAM, class V>
  static __device__ __forceinline__ V get(const T* p) {
    if (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    return *reinterpret_cast<const V*>(p);
  }
  __device__ __forceinline__ void drop_missing(unsigned there, int g) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!(there >> (16 * kt + 4 * g + e) & 1))
#pragma unroll
          for (int b = 0; b < VB; ++b) v[kt][e][b] = V4{};
  }
};

// The scales of the key at pool row `at` (1 where there is none).
__device__ __forceinline__ unsigned scale_byte(const MhaArgs& a, const uint8_t* scales, int hk, int at) {
  return at < 0 ? 127u : scales[scale_index(at, hk, a.Hkv, a.sh, a.ssh)];
}

// x as the sum of three bf16 numbers, exactly but for what lies 2^-24 below it and more (8 bits each,
// with the range of fp32, so no scales are needed; parts below 2^-126 the MFMA takes as zero; an infinity
// becomes NaN).
__device__ __forceinline__ void split3(float x0, float x1, bf16x2& h, bf16x2& m, bf16x2& l) {
  h = __builtin_convertvector(float2v{x0, x1}, bf16x2);
  const float r0 = x0 - (float)h[0], r1 = x1 - (float)h[1];
  m = __builtin_convertvector(float2v{r0, r1}, bf16x2);
  l = __builtin_convertvector(float2v{r0 - (float)m[0], r1 - (float)m[1]}, bf16x2);
}
struct Split8 {
  bf16x8 h, m, l;
  __device__ __forceinline__ void set(int i, float x0, float x1) {
    bf16x2 a, b, c;
    split3(x0, x1, a, b, c);
    h[i] = a[0], h[i + 1] = a[1];
    m[i] = b[0], m[i + 1] = b[1];
    l[i] = c[0], l[i + 1] = c[1];
  }
};
__device__ __forceinline__ floatx4 mfma_bf16(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A wave's queries as the MFMA's second operand, times log2(e)/√d_head: fp32 pieces of 4 columns, or
// for bf16 keys three bf16 parts of 8 columns.
template <class T, int DT, int RT>
struct Queries;
template <int DT, int RT>
struct Queries<float, DT, RT> {
  floatx4 q[RT][DT];
  __device__ __forceinline__ void load(const Rows<RT>& r, int dh, int g, float sl2) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < DT; ++c) {
        const int col = 16 * c + 4 * g;
        q[i][c] = r.q[i] && col < dh ? load4(r.q[i] + col) * sl2 : floatx4{0.f, 0.f, 0.f, 0.f};
      }
  }
};
template <int DT, int RT>
struct Queries<__bf16, DT, RT> {
  static constexpr int KC = (DT + 1) / 2;
  Split8 q[RT][KC];
  __device__ __forceinline__ void load(const Rows<RT>& r, int dh, int g, float sl2) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int col = 32 * c + 8 * g;
        floatx4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
        if (r.q[i] && col < dh) {
          x = load4(r.q[i] + col) * sl2;
          y = load4(r.q[i] + col + 4) * sl2;
        }
        q[i][c].set(0, x[0], x[1]);
        q[i][c].set(2, x[2], x[3]);
        q[i][c].set(4, y[0], y[1]);
        q[i][c].set(6, y[2], y[3]);
      }
  }
};

// Sᵀ tiles of 32 keys: st[r][kt][e] is key 16kt + 4g + e against row l16 of tile r.
template <int DT, int RT>
__device__ __forceinline__ void scores(const Keys32<float, DT>& x, const Queries<float, DT, RT>& q, int dh, int g,
                                       floatx4 (&st)[RT][2]) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
    for (int r = 0; r < RT; ++r) st[r][kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DT; ++c) {
      floatx4 k = x.k[kt][c];
      if (c >= DT - (DT > 4 ? 2 : 1) && 16 * c + 4 * g >= dh) k = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < RT; ++r) st[r][kt] = mfma16x16x4(k[e], q.q[r][c][e], st[r][kt]);
    }
  }
}
template <int DT, int RT>
__device__ __forceinline__ void scores(const Keys32<__bf16, DT>& x, const Queries<__bf16, DT, RT>& q, int dh, int g,
                                       floatx4 (&st)[RT][2]) {
  constexpr int KC = (DT + 1) / 2;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
    for (int r = 0; r < RT; ++r) st[r][kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      uint4v u = x.k[kt][c];
      if (32 * c + 8 * g >= dh) u = uint4v{0, 0, 0, 0};
      const bf16x8 k = __builtin_bit_cast(bf16x8, u);
#pragma unroll
      for (int r = 0; r < RT; ++r) st[r][kt] = mfma_bf16(k, q.q[r][c].l, st[r][kt]);
#pragma unroll
      for (int r = 0; r < RT; ++r) st[r][kt] = mfma_bf16(k, q.q[r][c].m, st[r][kt]);
#pragma unroll
      for (int r = 0; r < RT; ++r) st[r][kt] = mfma_bf16(k, q.q[r][c].h, st[r][kt]);
    }
  }
}

// acc += Vᵀ·Pᵀ.
template <int DT, int RT>
__device__ __forceinline__ void add_values(const Keys32<float, DT>& x, const floatx4 (&st)[RT][2], Sums<DT, RT>& s) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int b = 0; b < Sums<DT, RT>::VB; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int r = 0; r < RT; ++r) s.acc[r][b][c] = mfma16x16x4(x.v[kt][e][b][c], st[r][kt][e], s.acc[r][b][c]);
}
template <int DT, int RT>
__device__ __forceinline__ void add_values(const Keys32<__bf16, DT>& x, const floatx4 (&st)[RT][2], Sums<DT, RT>& s) {
  // the MFMA's 8 keys of a lane group: 4g … 4g + 3 of both tiles of 16
  Split8 p[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      p[r].set(4 * kt, st[r][kt][0], st[r][kt][1]);
      p[r].set(4 * kt + 2, st[r][kt][2], st[r][kt][3]);
    }
#pragma unroll
  for (int b = 0; b < Sums<DT, RT>::VB; ++b)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4v u;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          u[2 * kt + i] = __builtin_amdgcn_perm(x.v[kt][2 * i + 1][b][c >> 1], x.v[kt][2 * i][b][c >> 1],
                                                c & 1 ? 0x07060302u : 0x05040100u);
      const bf16x8 v = __builtin_bit_cast(bf16x8, u);
#pragma unroll
      for (int r = 0; r < RT; ++r) s.acc[r][b][c] = mfma_bf16(v, p[r].l, s.acc[r][b][c]);
#pragma unroll
      for (int r = 0; r < RT; ++r) s.acc[r][b][c] = mfma_bf16(v, p[r].m, s.acc[r][b][c]);
#pragma unroll
      for (int r = 0; r < RT; ++r) s.acc[r][b][c] = mfma_bf16(v, p[r].h, s.acc[r][b][c]);
    }
}

// Scores that a row does not see become −∞.
template <int RT>
__device__ __forceinline__ void mask(floatx4 (&st)[RT][2], const int (&vis)[RT], int x, unsigned there, int g) {
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = 16 * kt + 4 * g + e;
        if (x + key >= vis[r] || !(there >> key & 1)) st[r][kt][e] = -INFINITY;
      }
}

// The running softmax: scores to exp2(score − new maximum), sums rescaled.
template <int DT, int RT>
__device__ __forceinline__ void soften(floatx4 (&st)[RT][2], Sums<DT, RT>& s) {
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
      mx = fmaxf(mx, fmaxf(fmaxf(st[r][kt][0], st[r][kt][1]), fmaxf(st[r][kt][2], st[r][kt][3])));
    const float m_new = fmaxf(s.m[r], rows4_max(mx));
    const float at = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(s.m[r] - at);
    s.m[r] = m_new;
    float ps = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[r][kt][e] = __builtin_amdgcn_exp2f(st[r][kt][e] - at);
        ps += st[r][kt][e];
      }
    s.l[r] = s.l[r] * alpha + ps;
#pragma unroll
    for (int b = 0; b < Sums<DT, RT>::VB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) s.acc[r][b][c] *= alpha;
  }
}

// Of the lanes that have a row.
template <int DT, int RT>
__device__ __forceinline__ bool finite(const Sums<DT, RT>& s, bool live) {
  float z = 0.f;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    z += 0.f * s.l[r];
#pragma unroll
    for (int b = 0; b < Sums<DT, RT>::VB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) z += 0.f * s.acc[r][b][c][i];
  }
  return __ballot(live && z != 0.f) == 0;  // 0 times an infinity or NaN is NaN
}

// The sums of a wave's rows over keys x, x + stride, … again, where they came out as infinity or NaN (from
// such operands, or from a split into parts, which has no infinities):
// scores by the fp32 MFMA from whole operands, and every row adds the values of those keys alone that
// it sees (0 times an infinity that it does not see would be NaN).
__device__ __forceinline__ float number(float x) { return x; }
__device__ __forceinline__ float number(__bf16 x) { return (float)x; }
__device__ __forceinline__ float number(e4m3 x) { return __builtin_amdgcn_cvt_f32_fp8(x.bits, 0); }
// What an element of the key at pool row `at` is multiplied by.
template <class T>
__device__ __forceinline__ float key_scale(const MhaArgs& a, const uint8_t* scales, int hk, int at) {
  if (!std::is_same<T, e4m3>::value) return 1.f;
  const unsigned byte = scale_byte(a, scales, hk, at);
  return byte == 255 ? NAN : ldexpf(1.f, (int)byte - 127);  // (the conversions to bf16 and fp32 do as much)
}
template <class T, int DT, int RT>
__device__ void exact_sums(const MhaArgs& a, const Item& it, int row0, int x, int stride, Sums<DT, RT>& s) {
  constexpr int VB = Sums<DT, RT>::VB;
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  Rows<RT> rows;
  take_rows(a, it, row0, l16, rows);
  const T* kp = static_cast<const T*>(a.k) + (size_t)it.hk * a.dh;
  const T* vp = static_cast<const T*>(a.v) + (size_t)it.hk * a.dh;
  const size_t ld = (size_t)a.Hkv * a.dh;
  const float sl2 = a.scale * LOG2E;
  s.clear();
#pragma unroll 1
  for (; x < it.x1; x += stride) {
    const int at = row_of(a, it, x + (lane & 31), page_of(a, it.s, it.pre, x + (lane & 31)));
    const unsigned there = (unsigned)__ballot(at >= 0);
    floatx4 st[RT][2] = {};
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int key_at = __shfl(at, 16 * kt + l16, 64);
      const T* p = kp + (size_t)max(key_at, 0) * ld;
      const float ks = key_scale<T>(a, a.k_scale, it.hk, key_at);
#pragma unroll 1
      for (int c = 0; c < a.dh; c += 16) {
        const bool live = c + 4 * g < a.dh;
        floatx4 k = {0.f, 0.f, 0.f, 0.f};
        if (live) {
#pragma unroll
          for (int e = 0; e < 4; ++e) k[e] = number(p[c + 4 * g + e]) * ks;
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          floatx4 q = {0.f, 0.f, 0.f, 0.f};
          if (live && rows.q[r]) q = load4(rows.q[r] + c + 4 * g) * sl2;
#pragma unroll
          for (int e = 0; e < 4; ++e) st[r][kt] = mfma16x16x4(k[e], q[e], st[r][kt]);
        }
      }
    }
    mask<RT>(st, rows.vis, x, there, g);
    soften<DT, RT>(st, s);
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      const int row = __shfl(at, key, 64), from = (key & 12) * 4 + l16;
      if (row < 0) continue;
      const float vs = key_scale<T>(a, a.v_scale, it.hk, row);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const floatx4 pv = key < 16 ? st[r][0] : st[r][1];
        const float pe = (key & 2) ? ((key & 1) ? pv[3] : pv[2]) : ((key & 1) ? pv[1] : pv[0]);
        const float p = __shfl(pe, from, 64);
        const bool seen = x + key < rows.vis[r];
#pragma unroll
        for (int b = 0; b < VB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int col = 64 * b + 16 * g + 4 * i + c;
              if (seen && col < a.dh) s.acc[r][b][c][i] += p * (number(vp[(size_t)row * ld + col]) * vs);
            }
      }
    }
  }
}

// … of 16 rows from row0 on, each wave its own, over the item's keys; written out.
template <class T, int DT>
__device__ __forceinline__ void store_exact(const MhaArgs& a, const Item& it, int row0) {
  const int lane = threadIdx.x & 63, g = lane >> 4, row = row0 + (lane & 15);
  Sums<DT, 1> e;
  exact_sums<T, DT, 1>(a, it, row0, it.x0, STEP, e);
  const float L = rows4_sum(e.l[0]);
  if (row >= it.n_rows) return;
#pragma unroll
  for (int b = 0; b < Sums<DT, 1>::VB; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = 64 * b + 16 * g + 4 * j;
      if (col < a.dh)
        store(a, it, row, col, floatx4{e.acc[0][b][0][j], e.acc[0][b][1][j], e.acc[0][b][2][j], e.acc[0][b][3][j]}, e.m[0], L);
    }
}

// ---------------------------------------------------------------- few rows: keys through the registers

// Up to 16 rows an item.  Each of the block's 4 waves takes every fourth group of 32 keys and keeps its own
// running maximum and sum; the waves are joined through LDS in their order.  K and V are 16-byte loads into
// the registers that feed the MFMA: Sᵀ = K·Qᵀ takes consecutive columns of a key per lane, its result is, as
// it lies, the other operand of Oᵀ += Vᵀ·Pᵀ, and there a lane's 4 consecutive columns of V are rows of four
// MFMAs (row r of MFMA c is column 4r + c), so V needs no transposition and nothing passes through LDS on
// the way.  fp32 keys go into the fp32 MFMA; bf16 keys into the bf16 one with Q and P as three bf16 parts,
// which keep 2^-24 of each.  A wave's next K is under way while it works, its V from the scores on.  Bound
// by the reading with the MFMA's cycles in between: 64 sequences of 512 to 1024 keys (768 on average), 16
// K/V heads of 64, 4 rows each: 56 µs in bf16 (3.7 TB/s), 92 in fp32 (4.5 TB/s); with 1024 keys each 62 µs
// in bf16 (4.3 TB/s), 43 in e4m3 (3.1 TB/s).  On widened keys the fp32 MFMA took bf16's own keys of 64 such sequences 160 µs in a
// first version, the bf16 one 60.
template <int DT>
__device__ bool byte_sums(const MhaArgs& a, const Item& it, int x, int stride, int page, Sums<DT, 1>& s);  // e4m3 keys

template <int DT>
struct RowsLds {
  static constexpr int R = 16, OS = 64 * ((DT + 3) / 4) + 4;
  float m[NW][R], l[NW][R];
  __attribute__((aligned(16))) float o[NW][R][OS];
};
template <class T, int DT>
__device__ __forceinline__ void rows_item(const MhaArgs& a, RowsLds<DT>& lds) {
  constexpr int VB = Sums<DT, 1>::VB, RT = 1, R = RowsLds<DT>::R, STRIDE = STEP * NW;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int g = lane >> 4, l16 = lane & 15, k32 = lane & 31;

  Item it;
  int page;
  if (!take_item<T, R>(a, it, STEP * w + k32, page)) return;
  int x = it.x0 + STEP * w;
  Sums<DT, RT> s;
  s.clear();
  if constexpr (sizeof(T) == 1) {
    if (x < it.x1) {
      const bool good = byte_sums<DT>(a, it, x, STRIDE, page, s);
      if (!good) exact_sums<T, DT, RT>(a, it, it.row0, x, STRIDE, s);
    }
  } else if (x < it.x1) {
    Keys32<T, DT> keys;
    int at = row_of(a, it, x + k32, page);
    keys.template load_k<true>(a, it.hk, at, g, l16);
    Rows<RT> rows;
    take_rows(a, it, it.row0, l16, rows);
    Queries<T, DT, RT> q;
    q.load(rows, a.dh, g, a.scale * LOG2E);
    keys.template load_v<true>(a, it.hk, at, g, l16);
    page = page_of(a, it.s, it.pre, x + STRIDE + k32);
    for (; x < it.x1; x += STRIDE) {
      // the next keys' loads go out as soon as this step has used the registers
      const bool more = x + STRIDE < it.x1;
      const unsigned there = (unsigned)__ballot(at >= 0);
      floatx4 st[RT][2];
      scores(keys, q, a.dh, g, st);
      if (more) {
        at = row_of(a, it, x + STRIDE + k32, page);
        keys.template load_k<true>(a, it.hk, at, g, l16);
        page = page_of(a, it.s, it.pre, x + 2 * STRIDE + k32);
      }
      if (there != ~0u || x + STEP > rows.vmin) mask<RT>(st, rows.vis, x, there, g);
      soften(st, s);
      if (there != ~0u) keys.drop_missing(there, g);
      add_values(keys, st, s);
      if (more) keys.template load_v<true>(a, it.hk, at, g, l16);
    }
    if (!finite(s, it.row0 + l16 < it.n_rows)) exact_sums<T, DT, RT>(a, it, it.row0, it.x0 + STEP * w, STRIDE, s);
  }

  // Join the four waves in their order.
  s.l[0] = rows4_sum(s.l[0]);
  if (it.row0 + l16 < it.n_rows) {
    if (g == 0) {
      lds.m[w][l16] = s.m[0];
      lds.l[w][l16] = s.l[0];
    }
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<floatx4*>(&lds.o[w][l16][64 * b + 16 * g + 4 * j]) =
            floatx4{s.acc[0][b][0][j], s.acc[0][b][1][j], s.acc[0][b][2][j], s.acc[0][b][3][j]};
  }
  __syncthreads();
  const int n4 = a.dh / 4;
  for (int i = tid; i < R * n4; i += 64 * NW) {
    const int r = i / n4, c = 4 * (i - r * n4);
    if (it.row0 + r >= it.n_rows) break;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int j = 0; j < NW; ++j) M = fmaxf(M, lds.m[j][r]);
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NW; ++j) {
      const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(lds.m[j][r] - M);
      L += f * lds.l[j][r];
      o += f * *reinterpret_cast<const floatx4*>(&lds.o[j][r][c]);
    }
    store(a, it, it.row0 + r, c, o, M, L);
  }
}

// ---------------------------------------------------------------- single tokens: no matrix products

// The rows of one token: the query heads of a K/V head, all of which see the same keys.  Such items are
// bound by reading K and V; the MFMA of rows_item works on 16 rows whatever there are, and its cycles stand
// between the loads.  Vector instructions cost by the row.  64 sequences of 512 to 1024 keys (768 on
// average), 16 K/V heads of 64, µs by vectors and by the MFMA: 1 row 67 and 85 (5.9 TB/s), 2 rows 73 and 84,
// 4 rows 83 and 92; bf16 keys 1 row 40 and 53 (5.0 TB/s), 2 rows 43 and 54, 4 rows 55 and 56 (with a prefix
// of 2048 beside it 40 and 38): so 4 rows in fp32, 2 in bf16.  With 1024 keys each, by vectors: fp32 85 µs
// (6.3 TB/s), 88 and 94, bf16 48 µs (5.6 TB/s) and 49, e4m3 33 µs (4.0 TB/s) and 41.  e4m3 keys of 512 to 1024 (out of
// the chip's caches, which hold them) by vectors 24 and 31, by the MFMA 32 and 32, and 4 rows 43 against 33: so 2 rows
// in e4m3 as well.  LP lanes have a key's head, 16 bytes each (8 of e4m3), so that a load brings 64/LP whole keys;
// a score is added up over the LP lanes, l and the columns over the key groups once at the end, all of it in fp32.  While one half of the registers is in use, the
// loads of the other are under way, and the page of the step after them.
template <class T, int DT>
struct FewRows {
  static constexpr bool B8 = sizeof(T) == 1;
  static constexpr int E = B8 ? 8 : 16 / sizeof(T);       // columns of a lane
  using Piece = typename std::conditional<B8, float2v, floatx4>::type;
  static constexpr int N = (16 * DT + E - 1) / E;         // lanes of a head
  static constexpr int LP = N <= 2 ? 2 : N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : 32;
  static constexpr int KPI = 64 / LP;                     // keys of a load
  // loads of K, and of V, under way; as many are in use
  static constexpr int U = KPI > 16 || (B8 && KPI > 8) ? 64 / KPI : B8 ? 8 : 4;
  static constexpr int KEYS = U * KPI;                    // of a step; a lane finds the row of one
  static_assert(KEYS <= 64 && N <= 32, "a wave finds the rows of a step");
};
template <int R>
struct FewLds {
  float m[NW][R], l[NW][R];
  __attribute__((aligned(16))) float o[NW][R][128];
};
__device__ __forceinline__ void unpack(floatx4 x, float (&y)[4], float) {
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i];
}
__device__ __forceinline__ void unpack(floatx4 x, float (&y)[8], float) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = __uint_as_float(__float_as_uint(x[i]) << 16);
    y[2 * i + 1] = __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(float2v x, float (&y)[8], float scale) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2v p = __builtin_bit_cast(
        float2v, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(__float_as_uint(x[i / 2]), scale, true)
                       : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(__float_as_uint(x[i / 2]), scale, false));
    y[2 * i] = p[0];
    y[2 * i + 1] = p[1];
  }
}

template <class T, int DT, int R>
__device__ __forceinline__ void few_item(const MhaArgs& a, FewLds<R>& lds) {
  using G = FewRows<T, DT>;
  constexpr int E = G::E, LP = G::LP, U = G::U, KPI = G::KPI, KEYS = G::KEYS, STRIDE = NW * KEYS;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int part = lane % LP, kg = lane / LP;
  const bool live = E * part < a.dh;  // a lane of the group past the head is idle; its loads stay in range
  const int col = live ? E * part : a.dh - E;

  Item it;
  int page;
  if (!take_item<T, R>(a, it, KEYS * w + lane % KEYS, page)) return;
  const char* const kp = static_cast<const char*>(a.k) + ((size_t)it.hk * a.dh + col) * sizeof(T);
  const char* const vp = static_cast<const char*>(a.v) + ((size_t)it.hk * a.dh + col) * sizeof(T);
  const long long ld = (long long)a.Hkv * a.dh * sizeof(T);
  const float* qp = a.q + (size_t)it.tok0 * a.ld_q + (size_t)it.hk * a.G * a.dh + col;
  int x = it.x0 + KEYS * w;
  float m[R], l[R], acc[R][E];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[r][i] = 0.f;
  }
  if (x < it.x1) {
    using Piece = typename G::Piece;
    Piece k[2][U], v[2][U];
    unsigned k_scale[2] = {}, v_scale[2] = {};  // of the key that this lane finds
    unsigned long long there[2];
    auto load = [&](int b, int at) {
      there[b] = __ballot(at >= 0);
      if (G::B8) {
        k_scale[b] = scale_byte(a, a.k_scale, it.hk, at);
        v_scale[b] = scale_byte(a, a.v_scale, it.hk, at);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long o = max(__shfl(at, u * KPI + kg, 64), 0) * ld;
        if (G::B8) {  // a line may have other heads' parts: past the caches the reading took a sixth longer
          k[b][u] = *reinterpret_cast<const Piece*>(kp + o);
          v[b][u] = *reinterpret_cast<const Piece*>(vp + o);
        } else {
          k[b][u] = __builtin_nontemporal_load(reinterpret_cast<const Piece*>(kp + o));
          v[b][u] = __builtin_nontemporal_load(reinterpret_cast<const Piece*>(vp + o));
        }
      }
    };
    load(0, row_of(a, it, x + lane % KEYS, page));
    float q[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < E; ++i) q[r][i] = qp[(size_t)min(r, a.G - 1) * a.dh + i] * (a.scale * LOG2E);
    page = page_of(a, it.s, it.pre, x + STRIDE + lane % KEYS);
    // the keys of one half of the registers, while those of the other come
    auto step = [&](auto b) {
      constexpr int B = decltype(b)::value;
      if (x + STRIDE < it.x1) {
        load(1 - B, row_of(a, it, x + STRIDE + lane % KEYS, page));
        page = page_of(a, it.s, it.pre, x + 2 * STRIDE + lane % KEYS);
      }
      float s[R][U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float y[E];
        unpack(k[B][u], y, G::B8 ? scale_of(__shfl(k_scale[B], u * KPI + kg, 64)) : 1.f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float d = q[r][0] * y[0];
#pragma unroll
          for (int i = 1; i < E; ++i) d += q[r][i] * y[i];
          s[r][u] = aurlanes::group_reduce<1, LP, false>(live ? d : 0.f);
        }
      }
      if (there[B] != ~0ull) {  // keys that are not there: no score, and no value whatever lies in the row
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (!(there[B] >> (u * KPI + kg) & 1)) {
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][u] = -INFINITY;
            v[B][u] = Piece{};
          }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float mx = m[r];
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[r][u]);
        mx = aurlanes::group_reduce<LP, 64, true>(mx);
        const float at = mx == -INFINITY ? 0.f : mx, alpha = __builtin_amdgcn_exp2f(m[r] - at);
        m[r] = mx;
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[r][i] *= alpha;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[r][u] = __builtin_amdgcn_exp2f(s[r][u] - at);
          l[r] += s[r][u];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float y[E];
        unpack(v[B][u], y, G::B8 ? scale_of(__shfl(v_scale[B], u * KPI + kg, 64)) : 1.f);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < E; ++i) acc[r][i] += s[r][u] * y[i];
      }
      x += STRIDE;
    };
    for (;;) {
      step(std::integral_constant<int, 0>{});
      if (x >= it.x1) break;
      step(std::integral_constant<int, 1>{});
      if (x >= it.x1) break;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] = aurlanes::group_reduce<LP, 64, false>(l[r]);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[r][i] = aurlanes::group_sum_lanes<LP>(acc[r][i]);
    if (kg == 0 && live) {
#pragma unroll
      for (int i = 0; i < E; i += 4)
        *reinterpret_cast<floatx4*>(&lds.o[w][r][col + i]) = floatx4{acc[r][i], acc[r][i + 1], acc[r][i + 2], acc[r][i + 3]};
    }
    if (lane == 0) {
      lds.m[w][r] = m[r];
      lds.l[w][r] = l[r];
    }
  }
  __syncthreads();
  const int r = tid / 32, c = 4 * (tid % 32);
  if (r >= min(R, it.n_rows) || c >= a.dh) return;
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int j = 0; j < NW; ++j) M = fmaxf(M, lds.m[j][r]);
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(lds.m[j][r] - M);
    L += f * lds.l[j][r];
    o += f * *reinterpret_cast<const floatx4*>(&lds.o[j][r][c]);
  }
  store(a, it, r, c, o, M, L);
}

// ---------------------------------------------------------------- many rows: keys through LDS

// 16·NR·W rows an item, 16·NR of each of the block's W waves.  The block lays KT keys down in LDS as
// bf16 parts (fp32: three, whose six products above 2^-24 of the largest the MFMA sums; bf16 keys are
// one part, Q and P three), K as [key][column], V as [column][key], while the next keys' loads are
// under way: six bf16 products cost 6/16 of the fp32 MFMA's time for one.  Bound by the MFMA and by what
// lies between its issues, the conversion of the next tile and the softmax: 16 sequences of 259 to 503 tokens
// on a prefix of 4096, 16 heads of 64, fp32: 667 µs, 161 TFLOP/s (rows behind a sequence's last fill a fourth
// of its tiles; with 512 tokens each 696 µs, 210 TFLOP/s, the rate that a large library product of 1262 in
// bf16 leaves for six, and bf16 454 µs, 321 of 421).  The more rows, the less often K and V are loaded,
// converted and read from LDS: 16 rows a wave of 4 waves 1191 µs, of 8 waves 804, 32 rows a wave with the
// keys' places in LDS 667.  Tiles of 32x32 took 656 at d_head 64 and spilled more at 128.  (Of those here some
// spill at 256 registers too: fp32 keys of d_head 33 to 48 in 128 and 256 rows 18 and 9 registers, of d_head
// above 96 in 64 rows 12, others up to 4.)
template <class T, int DT, int W>
struct TileGeo {
  static constexpr bool F32 = std::is_same<T, float>::value;
  static constexpr int PARTS = F32 ? 3 : 1;
  static constexpr int KT = DT > 4 ? 32 : 64;      // keys of a tile
  static constexpr int KC = (DT + 1) / 2;          // 32-column steps of a score
  static constexpr int KROW = KC == 1 ? 64 : KC == 2 ? 128 : 256;
  static constexpr int KPLANE = KT * KROW, VPLANE = DT * 16 * KT * 2;
  static constexpr int TPR = 64 * W / KT, NI = (4 * KC + TPR - 1) / TPR;  // K: threads of a row, octets of a thread
  static constexpr int VC = F32 && 2 * DT * KT <= 64 * W ? 1 : 2, VN = 16 * DT / VC;  // V: VC columns of 8 keys a thread
  static_assert(VN * (KT / 8) <= 64 * W, "every piece of V has its thread");
};
// Granule q (16 bytes) of row r in rows of ROW bytes: every phase of 16 lanes covers the 64 banks once.
template <int ROW>
__device__ __forceinline__ int tile_granule(int r, int q) {
  return ROW == 64 ? split_granule(r, q) : ROW == 128 ? granule128(r, q) : r * 256 + ((q ^ r) & 15) * 16;
}
__device__ __forceinline__ float max3(float x, float y, float z) {  // one instruction; NaN if one is
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x, y), z);
}

template <class T, int DT, int W>
struct TileLds {
  using G = TileGeo<T, DT, W>;
  char k[G::PARTS * G::KPLANE], v[G::PARTS * G::VPLANE];
  long long offset[3][G::KT];  // in bytes, of the keys of this tile and the next two in the pools
  unsigned long long have[3];  // which of them are there
};
template <class T, int DT, int NR, int W>
__device__ __forceinline__ void tile_item(const MhaArgs& a, TileLds<T, DT, W>& lds) {
  using G = TileGeo<T, DT, W>;
  constexpr bool F32 = G::F32;
  constexpr int KT = G::KT, KC = G::KC, NI = G::NI, NK = KT / 16, VC = G::VC;
  char* const ks = lds.k;
  char* const vs = lds.v;
  constexpr unsigned long long ALL = KT == 64 ? ~0ull : 0xffffffffull;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int g = lane >> 4, l16 = lane & 15;

  Item it;
  int page;
  if (!take_item<T, 16 * NR * W>(a, it, tid % KT, page)) return;
  const int row0 = it.row0 + 16 * NR * w;  // this wave's
  Rows<NR> rows;
  take_rows(a, it, row0, l16, rows);
  int vmax = 0;
#pragma unroll
  for (int r = 0; r < NR; ++r) vmax = max(vmax, rows.vis[r]);
#pragma unroll
  for (int m = 1; m < 16; m *= 2) vmax = max(vmax, __shfl_xor(vmax, m, 64));

  // Where a tile's keys lie; the first KT threads ask for the pages' numbers a tile before they are needed.
  const long long ld = (long long)a.Hkv * a.dh * sizeof(T);
  int xp = it.x0 + tid;  // the key whose page is under way
  auto place = [&](int slot) {
    if (tid < KT) {
      const int at = row_of(a, it, xp, page);
      lds.offset[slot][tid] = at < 0 ? 0 : at * ld;
      const unsigned long long have = __ballot(at >= 0);
      if (tid == 0) lds.have[slot] = have;
      xp += KT;
      page = page_of(a, it.s, it.pre, xp);
    }
  };
  place(0);
  place(1);
  __syncthreads();

  const int kr = tid / G::TPR, ko = tid % G::TPR;  // K: row kr, octets ko + TPR·i
  const int vc = tid % G::VN * VC, vg = tid / G::VN;  // V: columns vc … of granule vg
  const bool v_on = vg < KT / 8;
  const int vkey = v_on ? 32 * (vg >> 2) + 4 * (vg & 3) : 0;  // … the keys vkey + 16·(i/4) + i%4
  const char* const kp = static_cast<const char*>(a.k) + (size_t)it.hk * a.dh * sizeof(T);
  const char* const vp = static_cast<const char*>(a.v) + ((size_t)it.hk * a.dh + min(vc, a.dh - VC)) * sizeof(T);
  floatx4 kx[NI][F32 ? 2 : 1];  // as loaded
  float vx[8][F32 ? VC : 1];    // bf16: a pair
  unsigned long long have = 0;  // of the keys in them
  auto load = [&](int slot) {
    have = lds.have[slot];
    const char* p = kp + lds.offset[slot][kr];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const char* q = p + min(8 * (ko + G::TPR * i), a.dh - 8) * (int)sizeof(T);
      kx[i][0] = *reinterpret_cast<const floatx4*>(q);
      if (F32) kx[i][F32] = *reinterpret_cast<const floatx4*>(q + 16);
    }
    if (G::VN * (KT / 8) < 64 * W && !v_on) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const char* q = vp + lds.offset[slot][vkey + 16 * (i >> 2) + (i & 3)];
      if (F32 && VC == 2) {
        const float2v x = *reinterpret_cast<const float2v*>(q);
        vx[i][0] = x[0];
        vx[i][F32 ? VC - 1 : 0] = x[1];
      } else {
        vx[i][0] = *reinterpret_cast<const float*>(q);
      }
    }
  };
  auto lay_down = [&] {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = ko + G::TPR * i;
      if (4 * KC % G::TPR != 0 && q >= 4 * KC) continue;
      const bool live = DT * 16 == 32 * KC || 8 * q < a.dh;
      char* p = ks + tile_granule<G::KROW>(kr, q);
      const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
      if (F32) {
        const floatx4 x = live ? kx[i][0] : zero, y = live ? kx[i][F32] : zero;
        Split8 s;
        s.set(0, x[0], x[1]);
        s.set(2, x[2], x[3]);
        s.set(4, y[0], y[1]);
        s.set(6, y[2], y[3]);
        *reinterpret_cast<bf16x8*>(p) = s.h;
        *reinterpret_cast<bf16x8*>(p + G::KPLANE) = s.m;
        *reinterpret_cast<bf16x8*>(p + 2 * G::KPLANE) = s.l;
      } else {
        *reinterpret_cast<floatx4*>(p) = live ? kx[i][0] : zero;
      }
    }
    if (G::VN * (KT / 8) < 64 * W && !v_on) return;
    if (have != ALL) {  // a key that is not there adds nothing, whatever lies in its place
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(have >> (vkey + 16 * (i >> 2) + (i & 3)) & 1))
#pragma unroll
          for (int c = 0; c < (F32 ? VC : 1); ++c) vx[i][c] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      char* p = vs + tile_granule<2 * KT>(vc + c, vg);
      if (F32) {
        Split8 s;
#pragma unroll
        for (int i = 0; i < 8; i += 2) s.set(i, vx[i][F32 ? c : 0], vx[i + 1][F32 ? c : 0]);
        *reinterpret_cast<bf16x8*>(p) = s.h;
        *reinterpret_cast<bf16x8*>(p + G::VPLANE) = s.m;
        *reinterpret_cast<bf16x8*>(p + 2 * G::VPLANE) = s.l;
      } else {
        uint4v u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          u[i] = __builtin_amdgcn_perm(__float_as_uint(vx[2 * i + 1][0]), __float_as_uint(vx[2 * i][0]),
                                       c ? 0x07060302u : 0x05040100u);
        *reinterpret_cast<uint4v*>(p) = u;
      }
    }
  };
  load(0);

  Queries<__bf16, DT, NR> q;
  q.load(rows, a.dh, g, a.scale * LOG2E);
  const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
  floatx4 acc[NR][DT];
  float m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[r][d] = zero;
  }

  auto compute = [&](int x, unsigned long long there, auto some) {
    floatx4 st[NR][NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      bf16x8 kf[G::PARTS][KC];
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int i = 0; i < G::PARTS; ++i)
          kf[i][c] = *reinterpret_cast<const bf16x8*>(ks + i * G::KPLANE + tile_granule<G::KROW>(16 * j + l16, 4 * c + g));
#pragma unroll
      for (int r = 0; r < NR; ++r) st[r][j] = zero;
      // products in ascending size
      auto add = [&](int part, auto of) {
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int r = 0; r < NR; ++r) st[r][j] = mfma_bf16(kf[part][c], of(q.q[r][c]), st[r][j]);
      };
      if (F32) add(F32 * 2, [](const Split8& s) { return s.h; });
      add(0, [](const Split8& s) { return s.l; });
      if (F32) {
        add(F32, [](const Split8& s) { return s.m; });
        add(F32, [](const Split8& s) { return s.h; });
      }
      add(0, [](const Split8& s) { return s.m; });
      add(0, [](const Split8& s) { return s.h; });
    }
    if (decltype(some)::value) {  // keys that some row does not see
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = 16 * j + 4 * g + e;
            if (x + key >= rows.vis[r] || !(there >> key & 1)) st[r][j][e] = -INFINITY;
          }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float mx = m[r];
#pragma unroll
      for (int j = 0; j < NK; ++j) mx = max3(max3(mx, st[r][j][0], st[r][j][1]), st[r][j][2], st[r][j][3]);
      const float m_new = rows4_max(mx);
      const float at = m_new == -INFINITY ? 0.f : m_new;
      if (__ballot(m_new != m[r])) {  // a maximum grew: rarely, after the first tiles
        const float alpha = __builtin_amdgcn_exp2f(m[r] - at);
        l[r] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[r][d] *= alpha;
      }
      m[r] = m_new;
      float ps = 0.f;
#pragma unroll
      for (int j = 0; j < NK; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          st[r][j][e] = __builtin_amdgcn_exp2f(st[r][j][e] - at);
          ps += st[r][j][e];
        }
      l[r] += ps;
    }
#pragma unroll
    for (int kk = 0; kk < KT / 32; ++kk) {
      Split8 pf[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int i = 0; i < 8; i += 2) pf[r].set(i, st[r][2 * kk + i / 4][i & 3], st[r][2 * kk + i / 4][(i & 3) + 1]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        bf16x8 vf[G::PARTS];
#pragma unroll
        for (int i = 0; i < G::PARTS; ++i)
          vf[i] = *reinterpret_cast<const bf16x8*>(vs + i * G::VPLANE + tile_granule<2 * KT>(16 * d + l16, 4 * kk + g));
        auto add = [&](int part, auto of) {
#pragma unroll
          for (int r = 0; r < NR; ++r) acc[r][d] = mfma_bf16(vf[part], of(pf[r]), acc[r][d]);
        };
        if (F32) add(F32 * 2, [](const Split8& s) { return s.h; });
        add(0, [](const Split8& s) { return s.l; });
        if (F32) {
          add(F32, [](const Split8& s) { return s.m; });
          add(F32, [](const Split8& s) { return s.h; });
        }
        add(0, [](const Split8& s) { return s.m; });
        add(0, [](const Split8& s) { return s.h; });
      }
    }
  };

  int slot = 0;
  for (int x = it.x0; x < it.x1; x += KT) {
    if (x > it.x0) __syncthreads();  // every wave is done with the last tile
    lay_down();
    const unsigned long long there = have;
    const int next = slot == 2 ? 0 : slot + 1;
    place(next == 2 ? 0 : next + 1);
    __syncthreads();
    if (x + KT < it.x1) load(next);
    slot = next;
    if (x >= vmax) continue;  // none of the wave's rows sees this tile
    if (there != ALL || x + KT > rows.vmin)
      compute(x, there, std::true_type{});
    else
      compute(x, there, std::false_type{});
  }

#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float z = 0.f * l[r];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (DT * 16 == a.dh || 16 * d + 4 * g + i < a.dh) z += 0.f * acc[r][d][i];
    const int row = row0 + 16 * r + l16;
    if (__ballot(row < it.n_rows && z != 0.f) == 0) {
      const float L = rows4_sum(l[r]);
      if (row < it.n_rows) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (DT * 16 == a.dh || 16 * d + 4 * g < a.dh) store(a, it, row, 16 * d + 4 * g, acc[r][d], m[r], L);
      }
    } else {
      store_exact<T, DT>(a, it, row0 + 16 * r);
    }
  }
}

#include "paged_attention_e4m3.hpp"

// The item of many rows, by the type of the pools.
template <class T, int DT, int W>
using ManyLds = typename std::conditional<sizeof(T) == 1, ByteLds<DT, W>, TileLds<T, DT, W>>::type;
template <class T, int DT, int NR, int W>
__device__ __forceinline__ void many_item(const MhaArgs& a, ManyLds<T, DT, W>& lds) {
  if constexpr (sizeof(T) == 1)
    byte_tile_item<DT, NR, W>(a, lds);
  else
    tile_item<T, DT, NR, W>(a, lds);
}

// ---------------------------------------------------------------- launches

// What a launch of 256-thread blocks holds: own items of 1, 2, 4 or 16 rows, prefix items of none, 16 or 64.
template <class T, int DT, int R, int PRE>
union StepLds {
  typename std::conditional<R == 16, RowsLds<DT>, FewLds<R>>::type own;
  typename std::conditional<PRE == 64, ManyLds<T, DT, NW>, typename std::conditional<PRE == 16, RowsLds<DT>, char>::type>::type pre;
};

// Waves a SIMD should hold.  bf16 keys leave registers for three, all but 2 to 19 that spill in 64-row items of
// d_head 33 to 64.  µs with three and with two, 16 heads: 100 sequences on a prefix of 8192, d_head 64 39.6 and
// 43.5; 30 of 32 heads on 8, prefix 4096 19.7 and 21.9; 64 on 32768 82 and 77.6, without own keys 48.6 and 51;
// of d_head 48 on 16384 63.2 and 61.6; tails of 30 to 60 tokens on 2048 51.4 and 49.5.  e4m3 keys, whose tiles wait
// in registers as bytes beside two parts of Q, want two: 64 on 32768 94 and 64, without own keys, out of the chip's
// caches, 48 and 50.
template <class T, int DT, int NR>
constexpr int kWaves = sizeof(T) == 2 && DT <= 4 && NR == 1 ? 3 : 2;

template <class T, int DT, int NR, int W>
__global__ void __launch_bounds__(64 * W, (kWaves<T, DT, NR>)) paged_mha_tile_kernel(MhaArgs a) {
  __shared__ __attribute__((aligned(1024))) ManyLds<T, DT, W> lds;
  many_item<T, DT, NR, W>(a, lds);
}

// A decode step of many sequences in one launch: the prefix's items, bound by their products, beside the
// own ones, bound by memory (64 sequences of 516 to 1018 keys on a prefix of 32768, 16 heads of 64, bf16: 80
// µs with the join, 91 in two launches; 48 sequences of 350 to 692, 4 heads of 128 on 4999: 46 and 58).  fp32
// heads of more than 96 columns spill 13 to 17 of 256 registers in most forms of it.
template <class T, int DT, int R, int PRE>
__global__ void __launch_bounds__(64 * NW, (PRE == 64 ? kWaves<T, DT, 1> : 2)) paged_mha_step_kernel(MhaArgs a) {
  __shared__ __attribute__((aligned(1024))) StepLds<T, DT, R, PRE> lds;
  if (PRE > 0 && (int)blockIdx.x < a.p_items) {
    if constexpr (PRE == 64) many_item<T, DT, 1, NW>(a, lds.pre);
    if constexpr (PRE == 16) rows_item<T, DT>(a, lds.pre);
    return;
  }
  if constexpr (R < 16)
    few_item<T, DT, R>(a, lds.own);
  else
    rows_item<T, DT>(a, lds.own);
}

// Own items of R rows, prefix items of 16, 64 or none.
template <class T, int DT, int R>
void launch_step(const MhaArgs& a, int p_tile, unsigned items, hipStream_t st) {
  auto* step = p_tile == 64 ? paged_mha_step_kernel<T, DT, R, 64> : paged_mha_step_kernel<T, DT, R, 0>;
  if constexpr (R < 16)
    if (p_tile == 16) step = paged_mha_step_kernel<T, DT, R, 16>;
  hipLaunchKernelGGL(step, dim3(items), dim3(256), 0, st, a);
}

// p_tile 0: items of one kind (or of one tile).
template <class T, int DT>
void launch_tile(const MhaArgs& a, int p_tile, int tile, int rows, unsigned items, hipStream_t st) {
  const dim3 g(items);
  const dim3 four(256);
  if (tile == 16) {
    if (rows == 1) return launch_step<T, DT, 1>(a, p_tile, items, st);
    if (rows == 2) return launch_step<T, DT, 2>(a, p_tile, items, st);
    if constexpr (std::is_same<T, float>::value)
      if (rows == 4) return launch_step<T, DT, 4>(a, p_tile, items, st);
    launch_step<T, DT, 16>(a, p_tile, items, st);
  } else if (tile == 64) {
    hipLaunchKernelGGL((paged_mha_tile_kernel<T, DT, 1, 4>), g, four, 0, st, a);
  } else if constexpr (DT > 4) {
    hipLaunchKernelGGL((paged_mha_tile_kernel<T, DT, 1, 8>), g, dim3(512), 0, st, a);
  } else if (tile == 128) {
    hipLaunchKernelGGL((paged_mha_tile_kernel<T, DT, 2, 4>), g, four, 0, st, a);
  } else {
    hipLaunchKernelGGL((paged_mha_tile_kernel<T, DT, 2, 8>), g, dim3(512), 0, st, a);
  }
}

template <class T>
void launch_head(const MhaArgs& a, int p_tile, int tile, int rows, unsigned items, hipStream_t st) {
  switch (head_tiles(a.dh)) {
    case 1: return launch_tile<T, 1>(a, p_tile, tile, rows, items, st);
    case 2: return launch_tile<T, 2>(a, p_tile, tile, rows, items, st);
    case 3: return launch_tile<T, 3>(a, p_tile, tile, rows, items, st);
    case 4: return launch_tile<T, 4>(a, p_tile, tile, rows, items, st);
    case 6: return launch_tile<T, 6>(a, p_tile, tile, rows, items, st);
    default: return launch_tile<T, 8>(a, p_tile, tile, rows, items, st);
  }
}

}  // namespace
