// Items of 16 rows and more on pools of e4m3: what is included by paged_attention.hpp.
//
// An e4m3 number is an fp16 one, so K and V go into the fp16 MFMA as they are, and queries and weights as two
// fp16 parts, both rounded to nearest: their error is at most 2^-23 of a number, one unit in fp32's last place, where
// the three bf16 parts of the bf16 pools leave 2^-24 for a product more.  (Numbers below 2^-11 of the row's largest
// are kept to 2^-34 of that.)  Parts cut toward zero left 2^-21, all on one side.  Bound by
// the softmax's instructions and the MFMA's between them: 16 sequences of 512 tokens on a prefix of 4096, 16 heads
// of 64, 310 us, 350 TFLOP/s of the 600 that a large library product's rate leaves for two (the first form, of three
// bf16 products and two barriers a tile, 478); a step of 64 sequences of 512 to 1024 keys on 32768, 16 heads of 64,
// 64 us, 50 of them for the prefix.  The weights' sums as products with ones: 4 us more, d_head 128 17 of 337.
//   * Scales.  Relative to the largest scale 2^E seen so far, of K and of V, a key's scale is 2^(e − E + kUp), which
//     the conversion to fp16 multiplies by: 448 times the largest one's is near fp16's end, and down to e − E =
//     −kSpread, where the smallest e4m3 number is the smallest fp16 one, that is exact.  E goes into the factor of
//     the scores, and into the sums when it grows.  A smaller scale leaves the item to exact_sums (50 times slower);
//     but 2^-117 and less (what zeros get) counts as 0 beside 2^-67 and more.
//   * Queries times 2^a with the row's largest between 2^12 and 2^13; a goes into the factor of the scores.
//   * Weights are exp2(score − m) for a reference m 14 below the row's maximum, so up to 2^14: their second part is
//     then 2^-38 of the largest or better.
#pragma once

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kUp = 7, kSpread = 15 + kUp;
constexpr int kLeastScale = 10;   // byte of 2^-117, the least that an append gives
constexpr int kNothing = 60;      // byte of 2^-67: beside it such ones are 2^-30 of its smallest number at most
constexpr float kAbove = 14.f;    // log2 of the largest weight
// Sums that leave no room for this factor below fp32's largest number are left to exact_sums, whose weights are at
// most 1: up to 96 ranges of four waves each are added up later.
constexpr float kRoom = 0x1p10f;

struct Halves8 {  // eight numbers in two fp16 parts; the second has what rounding to the first left
  f16x8 h, l;
  __device__ __forceinline__ void set(int i, float x0, float x1) {
    // A factor that the compiler does not know to be -1 leaves x - (float)h one instruction of mixed operands, where
    // it would take two (16 sequences of 512 tokens on 4096, 16 heads of 64: 310 us, 327 without).
    float minus;
    asm("s_mov_b32 %0, -1.0" : "=s"(minus));
    const f16x2 a = __builtin_convertvector(float2v{x0, x1}, f16x2);
    const float2v rest = {__builtin_fmaf((float)a[0], minus, x0), __builtin_fmaf((float)a[1], minus, x1)};
    const f16x2 b = __builtin_convertvector(rest, f16x2);
    h[i] = a[0], h[i + 1] = a[1];
    l[i] = b[0], l[i + 1] = b[1];
  }
};
__device__ __forceinline__ floatx4 mfma_f16(f16x8 a, f16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// The largest of m and the sizes of x; NaN if one is.
__device__ __forceinline__ float larger4(float m, floatx4 x) {
  return max3(max3(m, fabsf(x[0]), fabsf(x[1])), fabsf(x[2]), fabsf(x[3]));
}
// Four e4m3 numbers times a power of two as two pairs of fp16.
__device__ __forceinline__ uint2v widen4(unsigned x, float scale) {
  return uint2v{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, false)),
                __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, true))};
}

// Largest scales so far, as bytes; the same in all lanes.
struct Reference {
  int k, v;
  static __device__ __forceinline__ Reference none() { return {-2, -2}; }  // below a key's that is not there
};
// 2^(byte − of + kUp), and whether an item can go on with it (byte −1: there is no key, always).
__device__ __forceinline__ float relative(int byte, int of, bool& fits) {
  fits &= byte < 0 || (byte != 255 && (of - byte <= kSpread || (byte <= kLeastScale && of >= kNothing)));
  return scale_of((unsigned)max(127 + kUp + byte - of, 0));
}
// The larger of k and v bytes, each packed in 16 bits, over lanes 0 .. 63 (or of each half alike).
__device__ __forceinline__ unsigned wave_top(unsigned x) {
  typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
  auto up = [](unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, a), __builtin_bit_cast(ushort2v, b)));
  };
#pragma unroll
  for (int m = 1; m < 64; m *= 2) x = up(x, (unsigned)__shfl_xor((int)x, m, 64));
  return x;
}

// A wave's queries, and the power of two that undoes their scaling.
template <int DT, int RT>
struct HalfQueries {
  static constexpr int KC = (DT + 1) / 2;
  Halves8 q[RT][KC];
  int back[RT];
  float factor[RT];
  __device__ __forceinline__ void load(const Rows<RT>& r, int dh, int g, float sl2) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      floatx4 x[2 * KC];
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int col = 32 * c + 8 * g;
        x[2 * c] = x[2 * c + 1] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (r.q[i] && col < dh) {
          x[2 * c] = load4(r.q[i] + col);
          x[2 * c + 1] = load4(r.q[i] + col + 4);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(x[2 * c][e]), fabsf(x[2 * c + 1][e])));
      }
      top = rows4_max(top);
      // (an infinity or NaN stays one, and the sums show it)
      const int up = top > 0.f && top <= 3.402823466e38f ? 12 - ilogbf(top) : 0;
      back[i] = -up;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[2 * c + h][e] = ldexpf(x[2 * c + h][e], up) * sl2;
        q[i][c].set(0, x[2 * c][0], x[2 * c][1]);
        q[i][c].set(2, x[2 * c][2], x[2 * c][3]);
        q[i][c].set(4, x[2 * c + 1][0], x[2 * c + 1][1]);
        q[i][c].set(6, x[2 * c + 1][2], x[2 * c + 1][3]);
      }
    }
  }
  // The scores' factor for K relative to 2^(k − 127).
  __device__ __forceinline__ void relative_to(int k) {
#pragma unroll
    for (int i = 0; i < RT; ++i) factor[i] = fmaxf(ldexpf(1.f, back[i] + k - 127 - kUp), 1.17549435e-38f);
  }
};

// ---------------------------------------------------------------- up to 16 rows

// rows_item's ways for e4m3 keys: 32 keys of a wave's step in registers, 8 columns of K and 4 of V a lane.
// Lane l loads the scales of key l % 32; the others have them from there.
template <int DT>
struct Bytes32 {
  static constexpr int VB = (DT + 3) / 4, KC = (DT + 1) / 2;
  uint2v k[2][KC];
  unsigned v[2][4][VB];
  int k_scale, v_scale;  // bytes (where there is no key, row 0's)
  __device__ __forceinline__ void load_k(const MhaArgs& a, int hk, int at, int g, int l16) {
    const size_t ld = (size_t)a.Hkv * a.dh;
    const uint8_t* kp = static_cast<const uint8_t*>(a.k) + (size_t)hk * a.dh;
    const size_t s = scale_index(max(at, 0), hk, a.Hkv, a.sh, a.ssh);
    k_scale = a.k_scale[s];
    v_scale = a.v_scale[s];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint8_t* p = kp + (size_t)max(__shfl(at, 16 * kt + l16, 64), 0) * ld;
#pragma unroll
      for (int c = 0; c < KC; ++c) k[kt][c] = *reinterpret_cast<const uint2v*>(p + min(32 * c + 8 * g, a.dh - 8));
    }
  }
  __device__ __forceinline__ void load_v(const MhaArgs& a, int hk, int at, int g, int l16) {
    const size_t ld = (size_t)a.Hkv * a.dh;
    const uint8_t* vp = static_cast<const uint8_t*>(a.v) + (size_t)hk * a.dh;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint8_t* p = vp + (size_t)max(__shfl(at, 16 * kt + 4 * g + e, 64), 0) * ld;
#pragma unroll
        for (int b = 0; b < VB; ++b) v[kt][e][b] = *reinterpret_cast<const unsigned*>(p + min(64 * b + 4 * l16, a.dh - 4));
      }
  }
  __device__ __forceinline__ void drop_missing(unsigned there, int g) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!(there >> (16 * kt + 4 * g + e) & 1))
#pragma unroll
          for (int b = 0; b < VB; ++b) v[kt][e][b] = 0;
  }
};

// The sums of 16 rows over keys x, x + stride, … of the item; false where exact_sums has to make them.
template <int DT>
__device__ __forceinline__ bool byte_sums(const MhaArgs& a, const Item& it, int x, int stride, int page, Sums<DT, 1>& s) {
  constexpr int VB = Sums<DT, 1>::VB, KC = (DT + 1) / 2;
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15, k32 = lane & 31;
  Bytes32<DT> keys;
  int at = row_of(a, it, x + k32, page);
  keys.load_k(a, it.hk, at, g, l16);
  Rows<1> rows;
  take_rows(a, it, it.row0, l16, rows);
  HalfQueries<DT, 1> q;
  q.load(rows, a.dh, g, a.scale * LOG2E);
  keys.load_v(a, it.hk, at, g, l16);
  page = page_of(a, it.s, it.pre, x + stride + k32);
  Reference ref = Reference::none();
  bool fits = true;
  for (; x < it.x1; x += stride) {
    // the next keys' loads go out as soon as this step has used the registers
    const bool more = x + stride < it.x1;
    const unsigned there = (unsigned)__ballot(at >= 0);
    const int kb = at >= 0 ? keys.k_scale : -1, vb = at >= 0 ? keys.v_scale : -1;
    if (__ballot(kb > ref.k || vb > ref.v)) {  // a scale grew: rarely, after the first steps
      const unsigned top = __builtin_amdgcn_readfirstlane(wave_top((unsigned)max(kb, 0) << 16 | (unsigned)max(vb, 0)));
      const int k = max(ref.k, (int)(top >> 16)), v = max(ref.v, (int)(top & 0xffff));
      if (v != ref.v && ref.v >= 0) {
        const float less = ldexpf(1.f, ref.v - v);
#pragma unroll
        for (int b = 0; b < VB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) s.acc[0][b][c] *= less;
      }
      ref = Reference{k, v};
      q.relative_to(k);
    }
    const float ks = relative(kb, ref.k, fits), vs = relative(vb, ref.v, fits);
    floatx4 st[1][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const float scale = __shfl(ks, 16 * kt + l16, 64);
      st[0][kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint2v lo = widen4(keys.k[kt][c][0], scale), hi = widen4(keys.k[kt][c][1], scale);
        uint4v u = {lo[0], lo[1], hi[0], hi[1]};
        if (32 * c + 8 * g >= a.dh) u = uint4v{0, 0, 0, 0};
        const f16x8 k = __builtin_bit_cast(f16x8, u);
        st[0][kt] = mfma_f16(k, q.q[0][c].l, st[0][kt]);
        st[0][kt] = mfma_f16(k, q.q[0][c].h, st[0][kt]);
      }
    }
    if (more) {
      at = row_of(a, it, x + stride + k32, page);
      keys.load_k(a, it.hk, at, g, l16);
      page = page_of(a, it.s, it.pre, x + 2 * stride + k32);
    }
    if (there != ~0u || x + STEP > rows.vmin) mask<1>(st, rows.vis, x, there, g);
    // the running softmax
    float mx = fmaxf(fmaxf(fmaxf(st[0][0][0], st[0][0][1]), fmaxf(st[0][0][2], st[0][0][3])),
                     fmaxf(fmaxf(st[0][1][0], st[0][1][1]), fmaxf(st[0][1][2], st[0][1][3])));
    const float m_new = fmaxf(s.m[0], rows4_max(mx) * q.factor[0] - kAbove);
    const float ref_m = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(s.m[0] - ref_m);
    s.m[0] = m_new;
    float ps = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[0][kt][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[0][kt][e], q.factor[0], -ref_m));
        ps += st[0][kt][e];
      }
    s.l[0] = s.l[0] * alpha + ps;
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) s.acc[0][b][c] *= alpha;
    if (there != ~0u) keys.drop_missing(there, g);
    // acc += Vᵀ·Pᵀ; the MFMA's 8 keys of a lane group: 4g … 4g + 3 of both tiles of 16
    Halves8 p;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      p.set(4 * kt, st[0][kt][0], st[0][kt][1]);
      p.set(4 * kt + 2, st[0][kt][2], st[0][kt][3]);
    }
    uint2v vv[2][4][VB];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float scale = __shfl(vs, 16 * kt + 4 * g + e, 64);
#pragma unroll
        for (int b = 0; b < VB; ++b) vv[kt][e][b] = widen4(keys.v[kt][e][b], scale);
      }
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4v u;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            u[2 * kt + i] = __builtin_amdgcn_perm(vv[kt][2 * i + 1][b][c >> 1], vv[kt][2 * i][b][c >> 1],
                                                  c & 1 ? 0x07060302u : 0x05040100u);
        const f16x8 v = __builtin_bit_cast(f16x8, u);
        s.acc[0][b][c] = mfma_f16(v, p.l, s.acc[0][b][c]);
        s.acc[0][b][c] = mfma_f16(v, p.h, s.acc[0][b][c]);
      }
    if (more) keys.load_v(a, it.hk, at, g, l16);
  }
  const float back = ldexpf(1.f, ref.v - 127 - kUp);
#pragma unroll
  for (int b = 0; b < VB; ++b)
#pragma unroll
    for (int c = 0; c < 4; ++c) s.acc[0][b][c] *= back;
  float top = s.l[0];
#pragma unroll
  for (int b = 0; b < VB; ++b)
#pragma unroll
    for (int c = 0; c < 4; ++c) top = larger4(top, s.acc[0][b][c]);
  return __ballot(!fits || (it.row0 + l16 < it.n_rows && !(top * kRoom < INFINITY))) == 0;
}

// ---------------------------------------------------------------- many rows: keys through LDS

// tile_item's ways for e4m3 keys.  The block lays KT keys down in LDS as fp16, K as [key][column], V as
// [column][key], while the next keys' loads are under way: half of the waves K and half V, where that many have
// work, else all of them both.
template <int DT, int W>
struct ByteGeo {
  static constexpr int KT = 64, KC = (DT + 1) / 2;
  static constexpr int KROW = KC == 1 ? 64 : KC == 2 ? 128 : 256;
  static constexpr bool HALVES = DT <= W;
  static constexpr int KTHREADS = HALVES ? 32 * W : 64 * W;                       // K: threads …
  static constexpr int TPR = KTHREADS / KT, NI = (4 * KC + TPR - 1) / TPR;        // … of a row, octets of a thread
  static constexpr int VC = DT <= W / 2 ? 2 : 4, VN = 16 * DT / VC;               // V: VC columns of 8 keys a thread
  static_assert(VN * (KT / 8) <= KTHREADS, "every piece of V has its thread");
};
template <int DT, int W>
struct ByteLds {
  using G = ByteGeo<DT, W>;
  char k[2][G::KT * G::KROW], v[2][DT * 16 * G::KT * 2];  // of this tile and the next
  long long offset[3][G::KT];  // in bytes, of the keys of this tile and the next two in the pools
  unsigned long long have[3];  // which of them are there
  __attribute__((aligned(16))) float scale[3][2][G::KT];  // K's and V's, relative to …
  Reference ref[3];
};
template <int DT, int NR, int W>
__device__ __forceinline__ void byte_tile_item(const MhaArgs& a, ByteLds<DT, W>& lds) {
  using G = ByteGeo<DT, W>;
  constexpr int KT = G::KT, KC = G::KC, NI = G::NI, NK = KT / 16;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int g = lane >> 4, l16 = lane & 15;

  Item it;
  int page;
  if (!take_item<e4m3, 16 * NR * W>(a, it, tid % KT, page)) return;
  const int row0 = it.row0 + 16 * NR * w;  // this wave's
  Rows<NR> rows;
  take_rows(a, it, row0, l16, rows);
  int vmax = 0;
#pragma unroll
  for (int r = 0; r < NR; ++r) vmax = max(vmax, rows.vis[r]);
#pragma unroll
  for (int m = 1; m < 16; m *= 2) vmax = max(vmax, __shfl_xor(vmax, m, 64));

  // Where a tile's keys lie; the first wave asks for the pages' numbers a tile before they are needed, and lays
  // the scales down a tile after it asked for them, relative to the reference that this tile will have.
  Reference ref = Reference::none();
  bool fits = true;
  const long long ld = (long long)a.Hkv * a.dh;
  int xp = it.x0 + tid;  // the key whose page is under way
  int k_scale = -1, v_scale = -1;
  auto place = [&](int slot) {
    if (tid < KT) {
      const int last = slot == 0 ? 2 : slot - 1;
      Reference next = ref;
      if (__ballot(k_scale > ref.k || v_scale > ref.v)) {
        const unsigned top = __builtin_amdgcn_readfirstlane(wave_top((unsigned)max(k_scale, 0) << 16 | (unsigned)max(v_scale, 0)));
        next = Reference{max(ref.k, (int)(top >> 16)), max(ref.v, (int)(top & 0xffff))};
      }
      lds.scale[last][0][tid] = relative(k_scale, next.k, fits);
      lds.scale[last][1][tid] = relative(v_scale, next.v, fits);
      const int at = row_of(a, it, xp, page);
      const size_t s = scale_index(max(at, 0), it.hk, a.Hkv, a.sh, a.ssh);
      k_scale = a.k_scale[s];
      v_scale = a.v_scale[s];
      if (at < 0) k_scale = v_scale = -1;
      lds.offset[slot][tid] = at < 0 ? 0 : at * ld;
      const unsigned long long have = __ballot(at >= 0);
      if (tid == 0) {
        lds.have[slot] = have;
        lds.ref[last] = next;
      }
      xp += KT;
      page = page_of(a, it.s, it.pre, xp);
    }
  };
  place(0);
  place(1);
  __syncthreads();

  const bool k_on = !G::HALVES || tid < G::KTHREADS;
  const int kt = tid % G::KTHREADS, kr = kt / G::TPR, ko = kt % G::TPR;  // K: row kr, octets ko + TPR·i
  const int vt = G::HALVES ? tid - G::KTHREADS : tid;
  const bool v_on = vt >= 0 && vt < G::VN * (KT / 8);
  const int vc = v_on ? vt % G::VN * G::VC : 0, vg = v_on ? vt / G::VN : 0;  // V: columns vc … of granule vg
  const int vkey = 32 * (vg >> 2) + 4 * (vg & 3);                            // … the keys vkey + 16·(i/4) + i%4
  const uint8_t* const kp = static_cast<const uint8_t*>(a.k) + (size_t)it.hk * a.dh;
  const uint8_t* const vp = static_cast<const uint8_t*>(a.v) + (size_t)it.hk * a.dh + min(vc, a.dh - G::VC);
  uint2v kx[NI];  // as loaded
  unsigned vx[8];
  unsigned long long have = 0;  // of the keys in them
  auto load = [&](int slot) {
    have = lds.have[slot];
    if (k_on) {
      const uint8_t* p = kp + lds.offset[slot][kr];
#pragma unroll
      for (int i = 0; i < NI; ++i) kx[i] = *reinterpret_cast<const uint2v*>(p + min(8 * (ko + G::TPR * i), a.dh - 8));
    }
    if (v_on) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint8_t* p = vp + lds.offset[slot][vkey + 16 * (i >> 2) + (i & 3)];
        vx[i] = G::VC == 4 ? *reinterpret_cast<const unsigned*>(p) : *reinterpret_cast<const uint16_t*>(p);
      }
    }
  };

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
  load(0);
  HalfQueries<DT, NR> q;
  q.load(rows, a.dh, g, a.scale * LOG2E);

  auto lay_down = [&](int slot, int buffer) {
    char* const ks = lds.k[buffer];
    char* const vs = lds.v[buffer];
    const Reference next{__builtin_amdgcn_readfirstlane(lds.ref[slot].k), __builtin_amdgcn_readfirstlane(lds.ref[slot].v)};
    if (next.k != ref.k) q.relative_to(next.k);
    if (next.v != ref.v && ref.v >= 0) {
      const float less = ldexpf(1.f, ref.v - next.v);
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[r][d] *= less;
    }
    ref = next;
    if (k_on) {
      const float scale = lds.scale[slot][0][kr];
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int o = ko + G::TPR * i;
        if (4 * KC % G::TPR != 0 && o >= 4 * KC) continue;
        const uint2v lo = widen4(kx[i][0], scale), hi = widen4(kx[i][1], scale);
        *reinterpret_cast<uint4v*>(ks + tile_granule<G::KROW>(kr, o)) =
            DT * 16 == 32 * KC || 8 * o < a.dh ? uint4v{lo[0], lo[1], hi[0], hi[1]} : uint4v{0, 0, 0, 0};
      }
    }
    if (!v_on) return;
    if (have != ~0ull) {  // a key that is not there adds nothing, whatever lies in its place
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(have >> (vkey + 16 * (i >> 2) + (i & 3)) & 1)) vx[i] = 0;
    }
    const floatx4 s0 = *reinterpret_cast<const floatx4*>(&lds.scale[slot][1][vkey]),
                  s1 = *reinterpret_cast<const floatx4*>(&lds.scale[slot][1][vkey + 16]);
    unsigned x[8][2];  // pairs of columns
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint2v y = widen4(vx[i], i < 4 ? s0[i & 3] : s1[i & 3]);
      x[i][0] = y[0], x[i][1] = y[1];
    }
#pragma unroll
    for (int c = 0; c < G::VC; ++c) {
      uint4v u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        u[i] = __builtin_amdgcn_perm(x[2 * i + 1][c >> 1], x[2 * i][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
      *reinterpret_cast<uint4v*>(vs + tile_granule<2 * KT>(vc + c, vg)) = u;
    }
  };

  auto compute = [&](int x, unsigned long long there, int buffer, auto some) {
    const char* const ks = lds.k[buffer];
    const char* const vs = lds.v[buffer];
    floatx4 st[NR][NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      f16x8 kf[KC];
#pragma unroll
      for (int c = 0; c < KC; ++c)
        kf[c] = *reinterpret_cast<const f16x8*>(ks + tile_granule<G::KROW>(16 * j + l16, 4 * c + g));
#pragma unroll
      for (int r = 0; r < NR; ++r) st[r][j] = zero;
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int r = 0; r < NR; ++r) st[r][j] = mfma_f16(kf[c], q.q[r][c].l, st[r][j]);
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int r = 0; r < NR; ++r) st[r][j] = mfma_f16(kf[c], q.q[r][c].h, st[r][j]);
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
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < NK; ++j) mx = max3(max3(mx, st[r][j][0], st[r][j][1]), st[r][j][2], st[r][j][3]);
      const float m_new = __builtin_elementwise_maximum(m[r], rows4_max(mx) * q.factor[r] - kAbove);
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
          st[r][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r][j][e], q.factor[r], -at));
          ps += st[r][j][e];
        }
      l[r] += ps;
    }
#pragma unroll
    for (int kk = 0; kk < KT / 32; ++kk) {
      Halves8 pf[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int i = 0; i < 8; i += 2) pf[r].set(i, st[r][2 * kk + i / 4][i & 3], st[r][2 * kk + i / 4][(i & 3) + 1]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const f16x8 vf = *reinterpret_cast<const f16x8*>(vs + tile_granule<2 * KT>(16 * d + l16, 4 * kk + g));
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[r][d] = mfma_f16(vf, pf[r].l, acc[r][d]);
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[r][d] = mfma_f16(vf, pf[r].h, acc[r][d]);
      }
    }
  };

  // A tile is laid down by each wave as it is done with the last one: one barrier a tile, and the waves that
  // still work on the last one use the matrix cores meanwhile.
  lay_down(0, 0);
  place(2);
  __syncthreads();
  int slot = 0, buffer = 0;
  for (int x = it.x0; x < it.x1; x += KT) {
    const unsigned long long there = have;
    slot = slot == 2 ? 0 : slot + 1;
    const bool more = x + KT < it.x1;
    if (more) load(slot);
    if (x < vmax) {  // else none of the wave's rows sees this tile
      if (there != ~0ull || x + KT > rows.vmin)
        compute(x, there, buffer, std::true_type{});
      else
        compute(x, there, buffer, std::false_type{});
    }
    if (more) {
      buffer ^= 1;
      lay_down(slot, buffer);
      place(slot == 0 ? 2 : slot - 1);  // two tiles ahead: where the last one's places were
      __syncthreads();
    }
  }
  const bool exact = __syncthreads_or(!fits);
  const float back = ldexpf(1.f, ref.v - 127 - kUp);

#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float top = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (DT * 16 == a.dh || 16 * d + 4 * g < a.dh) top = larger4(top, acc[r][d]);
    const int row = row0 + 16 * r + l16;
    if (!exact && __ballot(row < it.n_rows && !(top * back * kRoom < INFINITY)) == 0) {
      const float L = rows4_sum(l[r]);
      if (row < it.n_rows) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (DT * 16 == a.dh || 16 * d + 4 * g < a.dh) store(a, it, row, 16 * d + 4 * g, acc[r][d] * back, m[r], L);
      }
    } else {
      store_exact<e4m3, DT>(a, it, row0 + 16 * r);
    }
  }
}
