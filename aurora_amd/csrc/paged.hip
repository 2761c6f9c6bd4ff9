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
  uint8_t *ks, *vs;  // scales of e4m3 pools, one for 2^ssh tokens of a head
  int ssh;
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

// ---------------------------------------------------------------- pools of e4m3

// A unit is a block of 2^ssh tokens of one head of K or V.  Its new values' largest size m gives the least scale
// 2^e, e from -117 to 119, with m <= 448·2^e: so all its numbers, subnormal ones too, are normal in bf16, and
// finite.  Where the block holds older tokens e is no less than before; if it grew, they are rounded once more.
// Elements are x·2^-e to the nearest e4m3, ties to even, and what lies beyond ±448·2^119 is that; an infinity or
// NaN is held as NaN and has no part in m.
//
// A unit's new tokens lie in registers between its maximum and its rounding, so the rows are read once: one wave
// holds up to 8 steps of 64 / LP tokens, LP lanes of 4 columns a head, and W = 4 waves share a unit that has more
// (up to 16 steps each).  Blocks walk over `chunk` rows of the batch each (no more than a block of tokens has, so
// that two of a sequence's units at most begin there) and take the units that begin in them, their last rows may lie
// behind.  16 prompts of 512 to 1024 tokens, 16 heads of 64, q rotated on the way: blocks of 32 tokens 55 us, 4.2 of
// the 5.1 TB/s of a large copy, of 64 and 128 62 and 58 (by two waves those of 64 59), of one 54 (312 while a wave
// took one block at a time); 8 heads of 128 take 66 to 76.  A step of 32 sequences: 6.5 us.
struct UnitArgs {
  int chunk, n_chunks, groups;  // rows of a chunk; blocks of a chunk, 4 / W units each
};

// Those prompts: a unit's steps issued one by one 59 us, two by two 61, one by one with seven waves on a SIMD, which
// spill 3 registers, 55; spans two by two 54, one by one 57.
constexpr int kUnitSteps = 8, kUnitAtOnce = 1, kAtOnce = 2;

// Four columns of a head, x, rotated with y, the ones that are their pairs' other halves, by t0 and t1, their (cos,
// sin): every product is rounded before the sum, so that a value next to the border of two e4m3 numbers falls
// where plain 32-bit arithmetic lets it fall.
__device__ __forceinline__ floatx4 rotated4(const AppendArgs& a, int col, floatx4 x, floatx4 y, floatx4 t0, floatx4 t1) {
#pragma clang fp contract(off)
  if (col >= a.rot) return x;
  if (a.pairs)
    return floatx4{x[0] * t0[0] - x[1] * t0[1], x[1] * t0[0] + x[0] * t0[1], x[2] * t0[2] - x[3] * t0[3],
                   x[3] * t0[2] + x[2] * t0[3]};
  const floatx4 c = {t0[0], t0[2], t1[0], t1[2]}, s = {t0[1], t0[3], t1[1], t1[3]};
  return col < a.rot / 2 ? x * c - y * s : x * c + y * s;
}

__device__ __forceinline__ unsigned round4(floatx4 x, int e) {  // of x·2^e
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = fabsf(x[i]) <= 3.402823466e38f ? __builtin_amdgcn_fmed3f(ldexpf(x[i], e), -448.f, 448.f) : NAN;
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
}

__device__ __forceinline__ unsigned again4(unsigned x, int e) {  // … of four e4m3 numbers
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
  return round4(floatx4{lo[0], lo[1], hi[0], hi[1]}, e);
}
// The largest size of the finite ones.
__device__ __forceinline__ float size4(floatx4 x) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(x[e]) <= 3.402823466e38f ? fabsf(x[e]) : 0.f);
  return m;
}
// The byte of the least scale for sizes up to m = f·2^x, f in [1, 2): 2^(x − 8), or 2^(x − 7) where f > 1.75.
__device__ __forceinline__ int scale_for(float m) {
  return min(max((int)((__float_as_uint(m) + 0x1fffffu) >> 23) - 8, 127 - 117), 127 + 119);
}

// LP lanes of a head, W waves of a unit, STEPS of each.
template <int LP, int W, int STEPS>
__device__ __forceinline__ void append_units(const AppendArgs& a, const UnitArgs& u, int block, float (&top)[4]) {
  constexpr int PER = 64 / LP;  // tokens of a wave's step
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int r0 = block / u.groups * u.chunk, r1 = min(r0 + u.chunk, a.b.n_tok);
  const int unit = block % u.groups * (4 / W) + w / W;
  const bool is_k = unit < a.Hkv, on = unit < 2 * a.Hkv;
  const int h = is_k ? unit : unit - a.Hkv, col = 4 * (lane % LP);
  const bool live = on && col < a.dh;
  const float* const src = (is_k ? a.k : a.v) + (size_t)h * a.dh;
  uint8_t* const pool = static_cast<uint8_t*>(is_k ? a.kp : a.vp) + (size_t)h * a.dh;
  const size_t ld = (size_t)a.Hkv * a.dh;
  const int S = 1 << a.ssh;
  for (int s = sequence_of(a.b, r0); s < a.b.b; ++s) {
    const Seq q = sequence(a.b, s);
    if (q.lo >= r1) break;
    const int past = q.len - q.n, first = max(0, -past);  // tokens before `first` have no place
    // the first unit that begins at row r0 or behind it
    int i = max(first, r0 - q.lo);
    if (i > first) i += -(past + i) & (S - 1);
    for (; i < q.n && q.lo + i < r1; i += S - ((past + i) & (S - 1))) {
      const int j = past + i, old = j & (S - 1), count = min(S - old, q.n - i);
      const int page = a.b.pages[(size_t)s * a.b.max_pages + (j >> a.sh)];
      if ((unsigned)page >= (unsigned)a.n_pages) continue;  // no page there: the rows are dropped
      const int row = (page << a.sh) + (j & ((1 << a.sh) - 1));
      uint8_t* const scale = (is_k ? a.ks : a.vs) + (on ? scale_index(row, h, a.Hkv, a.sh, a.ssh) : 0);
      const int held = old && on ? *scale : 0;
      floatx4 x[STEPS];
      float m = 0.f;
      // Lanes behind the head or the last token hold another's values: no branch stands between the loads.
      const int c = min(col, a.dh - 4), half = a.rot / 2;
      // where column c's partners and angles are (those of column 0 for a column that is not rotated)
      const bool turns = is_k && c < a.rot;
      const int cy = !turns || a.pairs ? c : c < half ? c + half : c - half;
      const int ct = !turns ? 0 : a.pairs ? c : 2 * (c < half ? c : c - half);
      auto place = [&](int n) { return min((n * W + w % W) * PER + lane / LP, count - 1); };
      auto take = [&](int n, floatx4 y) {
        x[n] = y;
        m = fmaxf(m, size4(y));
      };
      if (on) {
#pragma unroll
        for (int n0 = 0; n0 < STEPS; n0 += kUnitAtOnce)
          if (n0 * PER * W < count) {
            if (is_k && a.rot > 0) {
              floatx4 f[kUnitAtOnce], y[kUnitAtOnce], t0[kUnitAtOnce], t1[kUnitAtOnce];
#pragma unroll
              for (int n = 0; n < kUnitAtOnce; ++n) {
                const int k = place(n0 + n);
                const float* p = src + (size_t)(q.lo + i + k) * a.ld_kv;
                const float* tab = a.table + (size_t)(a.b.prefix_len + j + k) * a.rot + ct;
                f[n] = *reinterpret_cast<const floatx4*>(p + c);
                y[n] = *reinterpret_cast<const floatx4*>(p + cy);
                t0[n] = *reinterpret_cast<const floatx4*>(tab);
                t1[n] = *reinterpret_cast<const floatx4*>(a.pairs ? tab : tab + 4);
              }
#pragma unroll
              for (int n = 0; n < kUnitAtOnce; ++n) take(n0 + n, rotated4(a, c, f[n], y[n], t0[n], t1[n]));
            } else {
              floatx4 f[kUnitAtOnce];
#pragma unroll
              for (int n = 0; n < kUnitAtOnce; ++n)
                f[n] = *reinterpret_cast<const floatx4*>(src + (size_t)(q.lo + i + place(n0 + n)) * a.ld_kv + c);
#pragma unroll
              for (int n = 0; n < kUnitAtOnce; ++n) take(n0 + n, f[n]);
            }
          }
      }
#pragma unroll
      for (int o = 1; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o, 64));
      if constexpr (W > 1) {
        if (lane == 0) top[w] = m;
        __syncthreads();
        m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        __syncthreads();
      }
      const int byte = max(scale_for(m), held);
      if (live && old && byte > held)
        for (int k = (w % W) * PER + lane / LP; k < old; k += PER * W) {
          unsigned* p = reinterpret_cast<unsigned*>(pool + (size_t)(row - old + k) * ld + col);
          *p = again4(*p, held - byte);
        }
#pragma unroll
      for (int n = 0; n < STEPS; ++n) {
        const int k = (n * W + w % W) * PER + lane / LP;
        if (n * PER * W < count && live && k < count) *reinterpret_cast<unsigned*>(pool + (size_t)(row + k) * ld + col) = round4(x[n], 127 - byte);
      }
      if (on && lane == 0 && w % W == 0 && (!old || byte > held)) *scale = (uint8_t)byte;
    }
  }
}

// Blocks of fewer tokens than a step has (S·LP < 64): a wave takes STEPS whole steps of tokens, aligned to them,
// and every S·LP of its lanes have a block.  Lanes of a block's older tokens round those again.
template <int LP, int STEPS>
__device__ __forceinline__ void append_spans(const AppendArgs& a, const UnitArgs& u, int block) {
  constexpr int PER = 64 / LP, SPAN = PER * STEPS;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, S = 1 << a.ssh, group = LP << a.ssh;
  const int r0 = block / u.groups * u.chunk, r1 = min(r0 + u.chunk, a.b.n_tok);
  const int unit = block % u.groups * 4 + w;
  const bool is_k = unit < a.Hkv, on = unit < 2 * a.Hkv;
  const int h = is_k ? unit : unit - a.Hkv, col = 4 * (lane % LP), c = min(col, a.dh - 4);
  const float* const src = (is_k ? a.k : a.v) + (size_t)h * a.dh;
  uint8_t* const pool = static_cast<uint8_t*>(is_k ? a.kp : a.vp) + (size_t)h * a.dh;
  const size_t ld = (size_t)a.Hkv * a.dh;
  const int half = a.rot / 2;
  const bool turns = is_k && c < a.rot;
  const int cy = !turns || a.pairs ? c : c < half ? c + half : c - half;
  const int ct = !turns ? 0 : a.pairs ? c : 2 * (c < half ? c : c - half);
  for (int s = sequence_of(a.b, r0); s < a.b.b; ++s) {
    const Seq q = sequence(a.b, s);
    if (q.lo >= r1) break;
    const int past = q.len - q.n, first = max(0, -past);
    int i = max(first, r0 - q.lo);
    if (i > first) i += -(past + i) & (SPAN - 1);
    for (; i < q.n && q.lo + i < r1; i += SPAN - ((past + i) & (SPAN - 1))) {
      if (!on) continue;
      const int j = past + i, end = j + min(SPAN - (j & (SPAN - 1)), q.n - i), first_block = j >> a.ssh;
      const int j0 = (j & ~(SPAN - 1)) + lane / LP;  // the lane's token of the first step
#pragma unroll
      for (int n0 = 0; n0 < STEPS; n0 += kAtOnce) {
        if (j0 - lane / LP + n0 * PER >= end || j0 - lane / LP + (n0 + kAtOnce) * PER <= (first_block << a.ssh)) continue;
        floatx4 f[kAtOnce], y[kAtOnce], t0[kAtOnce], t1[kAtOnce];
        int page[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          const int at = min(max(j0 + (n0 + n) * PER, j), end - 1);  // (others' tokens where the lane has none)
          const float* p = src + (size_t)(q.lo + i + at - j) * a.ld_kv;
          f[n] = *reinterpret_cast<const floatx4*>(p + c);
          if (is_k && a.rot > 0) {
            const float* tab = a.table + (size_t)(a.b.prefix_len + at) * a.rot + ct;
            y[n] = *reinterpret_cast<const floatx4*>(p + cy);
            t0[n] = *reinterpret_cast<const floatx4*>(tab);
            t1[n] = *reinterpret_cast<const floatx4*>(a.pairs ? tab : tab + 4);
          }
          page[n] = a.b.pages[(size_t)s * a.b.max_pages + (at >> a.sh)];
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          const int at = j0 + (n0 + n) * PER;
          const floatx4 x = is_k && a.rot > 0 ? rotated4(a, c, f[n], y[n], t0[n], t1[n]) : f[n];
          const bool fresh = at >= j && at < end;
          float m = fresh ? size4(x) : 0.f;
          for (int o = 1; o < group; o *= 2) m = fmaxf(m, __shfl_xor(m, o, 64));
          // (a block lies in one page, that of its new tokens)
          const bool there = at >> a.ssh >= first_block && at >> a.ssh <= (end - 1) >> a.ssh &&
                             (unsigned)page[n] < (unsigned)a.n_pages;
          if (!there) continue;
          const int row = (page[n] << a.sh) + (at & ((1 << a.sh) - 1));
          uint8_t* const scale = (is_k ? a.ks : a.vs) + scale_index(row, h, a.Hkv, a.sh, a.ssh);
          const bool older = at >> a.ssh == first_block && (j & (S - 1));
          const int held = older ? *scale : 0, byte = max(scale_for(m), held);
          unsigned* const to = reinterpret_cast<unsigned*>(pool + (size_t)row * ld + c);
          if (col < a.dh && fresh)
            *to = round4(x, 127 - byte);
          else if (col < a.dh && at < j && byte > held)
            *to = again4(*to, held - byte);
          if (lane % group == 0 && (!older || byte > held)) *scale = (uint8_t)byte;
        }
      }
    }
  }
}

// A piece of q to a thread: the units of move(), whatever rows a block's pieces lie in.
__device__ __forceinline__ void rotate_q(const AppendArgs& a, int block) {
  const int per_rot = a.dh / 4 - (a.pairs ? 0 : a.rot / 8), per_row = a.H * per_rot;
  const long long first = (long long)block * 256;
  int t = (int)(first / per_row), u = (int)(first - (long long)t * per_row) + threadIdx.x;
  int s = sequence_of(a.b, t);  // of the block's first row
  t += u / per_row;
  u %= per_row;
  if (t >= a.b.n_tok) return;
  while (s < a.b.b && a.b.tok_off[s + 1] <= t) ++s;
  if (s >= a.b.b) return;  // a row behind the last sequence
  const Seq q = sequence(a.b, s);
  const int i = t - q.lo, j = q.len - q.n + i;
  if (i < 0 || i >= q.n || j < 0) return;
  const int h = u / per_rot;
  move(a, a.q + (size_t)t * a.ld_q + h * a.dh, a.q_out + (size_t)t * a.ld_qo + h * a.dh, u - h * per_rot,
       a.table + (size_t)(a.b.prefix_len + j) * a.rot, a.rot > 0);
}

// Blocks of the chunks' units, then those of q's rows.  W = 0: spans of small blocks.
template <int LP, int W, int STEPS>
__global__ void __launch_bounds__(256, STEPS > kUnitSteps ? 4 : 7) append_e4m3_kernel(AppendArgs a, UnitArgs u) {
  __shared__ float top[4];
  const int block = blockIdx.x, units = u.n_chunks * u.groups;
  if (block >= units)
    rotate_q(a, block - units);
  else if constexpr (W > 0)
    append_units<LP, W, STEPS>(a, u, block, top);
  else
    append_spans<LP, STEPS>(a, u, block);
}

template <int LP>
void launch_e4m3_lanes(const AppendArgs& a, const UnitArgs& u, int waves, int steps, unsigned blocks, hipStream_t st) {
  auto* kernel = append_e4m3_kernel<LP, 1, kUnitSteps>;
  if constexpr (LP < 64) {
    if (waves == 0) kernel = append_e4m3_kernel<LP, 0, kUnitSteps>;
  }
  if constexpr (LP >= 8) {  // 128 tokens of a block: LP·128 > 64·kUnitSteps
    if (waves == 4) kernel = append_e4m3_kernel<LP, 4, kUnitSteps>;
  }
  if constexpr (LP == 32) {
    if (waves == 4 && steps > kUnitSteps) kernel = append_e4m3_kernel<LP, 4, 2 * kUnitSteps>;
  }
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, a, u);
}

int launch_e4m3(aur_ctx* ctx, const char* who, const AppendArgs& a) {
  int lp = 2;
  while (4 * lp < a.dh) lp *= 2;
  const int S = 1 << a.ssh, waves = S * lp < 64 ? 0 : S * lp > 64 * kUnitSteps ? 4 : 1;
  const int steps = waves ? S * lp / (64 * waves) : kUnitSteps, run = waves ? S : 64 / lp * kUnitSteps;
  UnitArgs u;
  u.chunk = a.b.max_tok < run ? a.b.max_tok : run;
  u.n_chunks = (a.b.n_tok + u.chunk - 1) / u.chunk;
  u.groups = (2 * a.Hkv * (waves ? waves : 1) + 3) / 4;
  const int per_rot = a.dh / 4 - (a.pairs ? 0 : a.rot / 8);
  const uint64_t blocks = (uint64_t)u.n_chunks * u.groups + ((uint64_t)a.b.n_tok * a.H * per_rot + 255) / 256;
  if (blocks > kMaxBlocks) return aur::set_error(ctx, AUR_ELIMIT, "%s: n_tok=%d rows of %d heads", who, a.b.n_tok, a.H);
  auto* launch = lp == 2    ? launch_e4m3_lanes<2>
                 : lp == 4  ? launch_e4m3_lanes<4>
                 : lp == 8  ? launch_e4m3_lanes<8>
                 : lp == 16 ? launch_e4m3_lanes<16>
                            : launch_e4m3_lanes<32>;
  launch(a, u, waves, steps, (unsigned)blocks, ctx->stream);
  AUR_LAUNCH_CHECK(ctx, "append_e4m3_kernel");
  return 0;
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
  if (c->dtype != AUR_PAGED_F32 && c->dtype != AUR_PAGED_BF16 && c->dtype != AUR_PAGED_E4M3)
    return set_error(ctx, AUR_EINVAL, "%s: dtype %u", who, c->dtype);
  if (c->n_pages == 0 || c->page_len == 0 || (c->page_len & (c->page_len - 1)) || c->n_kv_head == 0 || c->d_head == 0)
    return set_error(ctx, AUR_EINVAL, "%s: n_pages=%u page_len=%u (a power of two) n_kv_head=%u d_head=%u", who,
                     c->n_pages, c->page_len, c->n_kv_head, c->d_head);
  if (c->d_head % 8 != 0 || c->d_head > 128)
    return set_error(ctx, AUR_ELIMIT, "%s: d_head=%u (multiples of 8 up to 128)", who, c->d_head);
  if ((uint64_t)c->n_pages * c->page_len > 0x7fffffffu || c->n_kv_head > 4096)
    return set_error(ctx, AUR_ELIMIT, "%s: pool of %u pages of %u rows, n_kv_head=%u", who, c->n_pages, c->page_len,
                     c->n_kv_head);
  if (c->dtype == AUR_PAGED_E4M3) {
    if (!c->k_scale || !c->v_scale || c->scale_len == 0 || (c->scale_len & (c->scale_len - 1)) ||
        c->scale_len > c->page_len)
      return set_error(ctx, AUR_EINVAL, "%s: scale_len=%u (a power of two up to page_len=%u) with both scales", who,
                       c->scale_len, c->page_len);
    if (c->scale_len > 128) return set_error(ctx, AUR_ELIMIT, "%s: scale_len=%u (up to 128)", who, c->scale_len);
  }
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
  if (cache->dtype == AUR_PAGED_E4M3) {
    a.ks = cache->k_scale; a.vs = cache->v_scale; a.ssh = log2_of(cache->scale_len);
    return launch_e4m3(ctx, who, a);
  }
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
