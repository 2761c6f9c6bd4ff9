// The next token of each row of logits, from a random number that the caller gives.
//
// With m the row's largest logit, a token's weight is w = exp((x − m) / T).  In the order of
// falling logits, equal ones by rising index, the kept tokens are a first part of the row: the
// first top_k; of these the fewest whose weight reaches top_p of the first top_k's; of these
// the ones with w >= min_p; the first one always.  The token is the least index i at which the
// sum of the kept weights up to it, in the order of the indexes, exceeds u times their sum.
//
// Whether a token is kept, and which one is drawn, hangs on sums that pass a border, so these
// have to come out the same in any order: a weight is computed in 64 bits (2^y = 2^n·e^r, |r| <=
// ln 2 / 2, twelve terms of e^r's series, to 2^-47) and held as a whole number of units of 2^-F,
// F = 63 − ⌈log2 vocab⌉ up to 50, so that a row's sum stays below 2^63.  Whole numbers add up
// exactly, which lets threads and atomics add them as they come.
//
// A block has one row, in LDS up to kStaged logits.  The border of top_k or top_p is found by one
// histogram over 1024 equal ranges of logits below m (each range's count or weight), a scan over
// it, and the exact order among the tokens of the one range that holds the border.  Where more
// than kList tokens lie in it, it is cut into 1024 again; a range of one value alone is cut by index.
// Where top_k leaves few tokens, those are compared with each other instead.
#include "common.hpp"
#include "lanes.hpp"
#include "sample_ranges.hpp"

#include <cmath>

using namespace aursample;

namespace {

typedef unsigned long long u64;
typedef unsigned uint32;

struct SampleArgs {
  const float *logits, *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* tokens;
  float* logprob;
  int vocab, ld, frac;  // weights in units of 2^-frac
  // Of rows that several blocks share, of each segment: the largest logit, the weight of what min_p keeps (for
  // each of kParts parts of it), and the histograms (of counts for top_k).
  int segments;
  float* seg_max;
  u64 *seg_mass, *mass;
  uint32* count;
};

typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kList = 1024, kPairs = 64;
constexpr int kSuper = 8;          // chunks whose weights are added up together
constexpr int kMaxVocab = 1 << 20;
constexpr int kStaged = 32768;     // logits of a row in LDS
constexpr int kSegment = 16384;    // … of a block, where several share a row
constexpr int kMaxSegments = kMaxVocab / kSegment;
constexpr int kParts = 4;          // of a segment: chunks of the block that goes through the row at last

struct Entry {
  float x;
  int i;
  u64 w;
};

struct SampleLds {
  u64 hist[kBins];
  __attribute__((aligned(16))) Entry list[kList], pairs[kPairs];
  u64 wave[kSuper * 16];
  u64 super[kMaxSegments];
  float red[16];
  u64 before, upto;
  int bin, count, best, token;
};

// Moves within a wave by DPP, 0 where there is no source lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp64(u64 x) {
  const uint32 lo = __builtin_amdgcn_update_dpp(0, (int)(uint32)x, CTRL, ROWS, 0xf, false);
  const uint32 hi = __builtin_amdgcn_update_dpp(0, (int)(uint32)(x >> 32), CTRL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 lane64(u64 x, int lane) {
  return (u64)(uint32)__builtin_amdgcn_readlane((int)(uint32)(x >> 32), lane) << 32 |
         (uint32)__builtin_amdgcn_readlane((int)(uint32)x, lane);
}
// The sum of the lanes up to this one: within rows of 16 lanes, then rows 0 and 2 to the next one, then the
// first half to the second.
__device__ __forceinline__ u64 wave_scan(u64 x) {
  x += dpp64<0x111, 0xf>(x);
  x += dpp64<0x112, 0xf>(x);
  x += dpp64<0x114, 0xf>(x);
  x += dpp64<0x118, 0xf>(x);
  x += dpp64<0x142, 0xa>(x);
  x += dpp64<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ u64 wave_sum(u64 x) { return lane64(wave_scan(x), 63); }
__device__ __forceinline__ u64 quad_sum(u64 x) {  // of four neighbouring lanes
  x += dpp64<0xb1, 0xf>(x);
  return x + dpp64<0x4e, 0xf>(x);
}

// The order of falling logits, equal ones by rising index.
__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

// The coefficients of 2^r's series from r^11 down to r.
struct Series {
  double c[11];
  __device__ __forceinline__ constexpr Series() : c{} {
    constexpr double l = 0.6931471805599453;
    double x = 1.0;
    for (int i = 1; i <= 11; ++i) c[11 - i] = x *= l / i;
  }
  // In registers, where the compiler would copy each one there from a constant in every use (32 rows of 32768, top_p:
  // 37 us, 42 without; the last kernel of wide rows has no registers left for them).
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int i = 0; i < 11; ++i) asm("" : "+v"(c[i]));
  }
};

// The weight of logit v in units of 2^-frac, to the nearest; scale is log2(e) / T.  No instruction of it runs at
// less than the rate of the others: conversions and powers of two are sums and moves of bits.
__device__ __forceinline__ u64 weight_of(float v, float m, double scale, int frac, const Series& s) {
  const double y = fmax(((double)v - (double)m) * scale, -2000.0);
  const double t = y + kWhole, r = y - (t - kWhole);  // 2^y = 2^n·2^r, |r| <= 1/2
  double p = s.c[0];
#pragma unroll
  for (int i = 1; i < 11; ++i) p = __builtin_fma(p, r, s.c[i]);
  p = __builtin_fma(p, r, 1.0);
  // times 2^(n + frac), at least 2^-2 (which rounds to nothing), to the nearest below 2^52
  const u64 up = (u64)(uint32)max(low32(t) + frac, -2) << 52;
  const double w = __longlong_as_double((long long)((u64)__double_as_longlong(p) + up)) + 0x1p52;
  return (u64)__double_as_longlong(w) & 0xfffffffffffffull;
}

// A row's filters, those that do nothing as values that say so (k = 0, p = 1, floor_y = −∞).
struct Filters {
  float T, p;
  int k;
  double floor_y;  // log min_p: kept tokens have (x − m) / T >= floor_y
  __device__ __forceinline__ Filters(const SampleArgs& a, int r) {
    T = a.temperature ? a.temperature[r] : 1.f;
    p = a.top_p ? a.top_p[r] : 1.f;
    if (!(p < 1.f)) p = 1.f;
    k = a.top_k ? a.top_k[r] : 0;
    if (k >= a.vocab || k < 0) k = 0;
    const float least_p = a.min_p ? a.min_p[r] : 0.f;
    floor_y = least_p > 0.f ? log((double)fminf(least_p, 1.f)) : -INFINITY;
  }
  // The least logit that min_p keeps of a row with the largest one m.
  __device__ __forceinline__ float least(float m) const {
    return floor_y == -INFINITY ? -INFINITY : least_kept(m, T, floor_y);
  }
  __device__ __forceinline__ bool greedy() const { return !(T > 0.f) || k == 1 || p <= 0.f; }
};

__device__ __forceinline__ u64 p_target(float p, u64 mass) { return (u64)fmax(ceil((double)p * (double)mass), 1.0); }

// One row of TH threads, in chunks of 4 * TH logits: in LDS (ROW > 0), or read again in each pass.
template <int TH, int ROW>
struct Row {
  static constexpr int NW = TH / 64;
  const SampleArgs& a;
  SampleLds& lds;
  floatx4* held;  // the row in LDS
  const float* x;
  int n_chunks;
  double scale, inv_t;  // log2(e) / T, 1 / T
  float m, T;
  Series series;
  bool infinite;  // the largest logit is +∞: such ones count as 0, all others as −∞

  __device__ __forceinline__ Row(const SampleArgs& a, SampleLds& lds, floatx4* held, int r)
      : a(a), lds(lds), held(held), x(a.logits + (size_t)r * a.ld), n_chunks((a.vocab + 4 * TH - 1) / (4 * TH)),
        infinite(false) {
    if (ROW > 0) series.keep();
  }
  __device__ __forceinline__ void take(float most, float t) {
    infinite = most == INFINITY;
    m = infinite ? 0.f : most;
    T = t;
    inv_t = 1.0 / (double)T;
    scale = 1.4426950408889634 / (double)T;
  }

  __device__ __forceinline__ floatx4 ordinary(floatx4 v) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] == INFINITY ? 0.f : -INFINITY;
    return v;
  }
  // Chunk c as it lies in memory (rows need not be aligned); −∞ behind the row.
  __device__ __forceinline__ floatx4 raw(int c) const {
    const int i = 4 * (c * TH + threadIdx.x);
    if (4 * TH * (c + 1) <= a.vocab) return *reinterpret_cast<const floatx4_any*>(x + i);
    floatx4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < a.vocab) v[e] = x[i + e];
    return v;
  }
  // N chunks from c on, their loads under way together.
  template <int N>
  __device__ __forceinline__ void raw(int c, floatx4 (&v)[N]) const {
    if (4 * TH * (c + N) <= a.vocab) {
      const floatx4_any* p = reinterpret_cast<const floatx4_any*>(x) + c * TH + threadIdx.x;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = p[i * TH];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = raw(c + i);
    }
  }
  // A logit that is NaN counts as −∞.
  __device__ __forceinline__ floatx4 clean(floatx4 v) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] == v[e] ? v[e] : -INFINITY;
    return infinite ? ordinary(v) : v;
  }
  // f(chunk, index of the first, four logits) for the chunks from c0 up to c1.
  template <class F>
  __device__ __forceinline__ void each(int c0, int c1, F f) const {
    if constexpr (ROW > 0) {
      for (int c = c0; c < c1; ++c) f(c, 4 * (c * TH + (int)threadIdx.x), held[c * TH + threadIdx.x]);
    } else {
      for (int c = c0; c < c1;) {  // four under way together
        floatx4 v[4];
        raw(c, v);
#pragma unroll 1
        for (int i = 0; i < 4 && c < c1; ++i, ++c) {
          f(c, 4 * (c * TH + (int)threadIdx.x), clean(v[0]));
          v[0] = v[1];
          v[1] = v[2];
          v[2] = v[3];
        }
      }
    }
  }

  // g(index, logit) of four logits.  A block that streams its row goes through much code once, and what it reads of
  // code costs it more than a loop over one copy of g does (64 rows of 131072: 94 us, with four copies 124, while
  // two lists and a segment's weights were made for each; 48 either way where the parts' sums spare those); a row in LDS is passed over by less (32 rows of 8192:
  // 10.9 us by four copies, 11.7 by one).
  template <class G>
  static __device__ __forceinline__ void one_by_one(floatx4 v, int i, G g) {
    if constexpr (ROW > 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) g(i + e, v[e]);
    } else {
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        g(i + e, v[0]);
        v = floatx4{v[1], v[2], v[3], v[0]};
      }
    }
  }
  __device__ __forceinline__ u64 weight(float v) const { return weight_of(v, m, scale, a.frac, series); }

  __device__ __forceinline__ float block_max(float v) {
    v = aurlanes::group_reduce<1, 64, true>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds.red[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) v = fmaxf(v, lds.red[w]);
    return v;
  }

  // The first index of logit v in the chunks from c0 up to c1.
  __device__ __forceinline__ int first_of(float v, int c0, int c1) {
    int token = 0x7fffffff;
    each(c0, c1, [&](int, int i, floatx4 y) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (y[e] == v) token = min(token, i + e);
    });
    __syncthreads();
    if (threadIdx.x == 0) lds.token = 0x7fffffff;
    __syncthreads();
    if (token != 0x7fffffff) atomicMin(&lds.token, token);
    __syncthreads();
    return lds.token;
  }

  // The entry of sums[0 .. n), n <= 128, at which they exceed r; r becomes what is left of it there.  `all` is
  // their sum.  Every wave finds it by itself.
  __device__ __forceinline__ int locate(const u64* sums, int n, u64& r) const {
    const int lane = threadIdx.x & 63;
    const u64 s0 = 2 * lane < n ? sums[2 * lane] : 0, s1 = 2 * lane + 1 < n ? sums[2 * lane + 1] : 0;
    const u64 up = wave_scan(s0 + s1) - s0 - s1;
    const bool here = up <= r && r < up + s0 + s1, second = r >= up + s0;
    const int at = __builtin_ctzll(__ballot(here));
    const u64 rest = lane64(r - up - (second ? s0 : 0), at);
    const int odd = (int)(__ballot(second) >> at & 1);
    r = rest;
    return 2 * at + odd;
  }
  __device__ __forceinline__ u64 sum_of(const u64* sums, int n) const {
    const int lane = threadIdx.x & 63;
    return wave_sum((2 * lane < n ? sums[2 * lane] : 0) + (2 * lane + 1 < n ? sums[2 * lane + 1] : 0));
  }
  // The weights f(index, logit) of the chunks from c0 up to c1, kSuper at most, added up by waves.
  template <class F>
  __device__ __forceinline__ void sum_waves(int c0, int c1, F f) {
    each(c0, c1, [&](int c, int i, floatx4 v) {
      u64 sum = 0;
      one_by_one(v, i, [&](int at, float x) { sum += f(at, x); });
      sum = wave_sum(sum);
      if ((threadIdx.x & 63) == 0) lds.wave[(c - c0) * NW + (threadIdx.x >> 6)] = sum;
    });
    __syncthreads();
  }
  // The least index at which the sum of the weights f(index, logit) up to it exceeds place(their sum).
  template <class F, class G>
  __device__ __forceinline__ int pick(F f, G place, u64& total) {
    const int n = (n_chunks + kSuper - 1) / kSuper;
    u64 r;
    int c0 = 0;
    __syncthreads();
    if (n == 1) {
      sum_waves(0, n_chunks, f);
      total = sum_of(lds.wave, n_chunks * NW);
      r = place(total);
    } else {
      for (int s = threadIdx.x; s < n; s += TH) lds.super[s] = 0;
      __syncthreads();
      for (int s = 0; s < n; ++s) {
        u64 sum = 0;
        each(s * kSuper, min((s + 1) * kSuper, n_chunks),
             [&](int, int i, floatx4 v) { one_by_one(v, i, [&](int at, float x) { sum += f(at, x); }); });
        sum = wave_sum(sum);
        if ((threadIdx.x & 63) == 0) atomicAdd(&lds.super[s], sum);
      }
      __syncthreads();
      total = sum_of(lds.super, n);
      r = place(total);
      c0 = locate(lds.super, n, r) * kSuper;
      sum_waves(c0, min(c0 + kSuper, n_chunks), f);
    }
    return pick_in(c0, min(c0 + kSuper, n_chunks), r, f);
  }
  // … at which what sum_waves added up from chunk c0 on exceeds r.
  template <class F>
  __device__ __forceinline__ int pick_in(int c0, int c1, u64 r, F f) {
    const int w = threadIdx.x >> 6;
    const int at = locate(lds.wave, (c1 - c0) * NW, r);
    if (w == at % NW)
      each(c0 + at / NW, c0 + at / NW + 1, [&](int, int i, floatx4 v) {
        u64 sum = 0;
        one_by_one(v, i, [&](int at, float x) { sum += f(at, x); });
        u64 up = wave_scan(sum) - sum;
        if (up <= r && r < up + sum)
          one_by_one(v, i, [&](int at, float x) {
            const u64 t = f(at, x);
            if (up <= r && r < up + t) lds.token = at;
            up += t;
          });
      });
    __syncthreads();
    return lds.token;
  }

  // Of the n <= kPairs entries in `list`, compared with each other, the one at which the sum of f(entry), in the
  // order of falling logits, rising indexes, reaches the target (which it does).  Four threads have an entry.
  template <class F>
  __device__ __forceinline__ Entry reach_in_pairs(const Entry* list, int n, u64 target, F f) {
    const int e = threadIdx.x >> 2;
    const Entry own = list[min(e, n - 1)];
    u64 ahead = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 3; j < n; j += 4) {
      const Entry o = list[j];
      ahead += before(o.x, o.i, own.x, own.i) ? f(o) : 0;
    }
    ahead = quad_sum(ahead);
    if (e < n && ahead < target && target <= ahead + f(own)) lds.best = e;
    __syncthreads();
    return list[lds.best];
  }
  // The same of the n <= kList entries in lds.list, all of them in one range: by kBins parts of it, or where one
  // part holds more than kPairs (many equal ones), all with each other.
  template <class F>
  __device__ __forceinline__ Entry reach_in_list(int n, u64 target, F f, const Ranges& ranges, int bin) {
    constexpr int PER = kList / TH;
    const int tid = threadIdx.x;
    if (n <= kPairs) return reach_in_pairs(lds.list, n, target, f);
    const Ranges part{ranges.hi - (bin - 0.5) / ranges.inv, ranges.inv * kBins};
    clear();
    int at[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      at[i] = -1;
      if (tid + TH * i < n) {
        const Entry e = lds.list[tid + TH * i];
        at[i] = max(part.of(e.x), 0);
        atomicAdd(&lds.hist[at[i]], f(e));
      }
    }
    __syncthreads();
    find(lds.hist, [&](u64) { return target; });
    const int here = lds.bin;
    const u64 rest = target - lds.before;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at[i] == here) {
        const int k = atomicAdd(&lds.count, 1);
        if (k < kPairs) lds.pairs[k] = lds.list[tid + TH * i];
      }
    __syncthreads();
    if (lds.count <= kPairs) return reach_in_pairs(lds.pairs, lds.count, rest, f);
    for (int i = tid; i < n; i += TH) {
      const Entry own = lds.list[i];
      u64 ahead = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) ahead += before(lds.list[j].x, lds.list[j].i, own.x, own.i) ? f(lds.list[j]) : 0;
      if (ahead < target && target <= ahead + f(own)) lds.best = i;
    }
    __syncthreads();
    return lds.list[lds.best];
  }
  // An empty histogram, list and answer.
  __device__ __forceinline__ void clear() {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBins / TH; ++i) lds.hist[threadIdx.x + TH * i] = 0;
    if (threadIdx.x == 0) lds.bin = -1, lds.count = 0;
    __syncthreads();
  }
  // The range at which the sum over the ranges reaches target(their sum), which is returned: lds.bin (left as it
  // is where there is none), the sums before it and with it lds.before and lds.upto.
  template <class W, class G>
  __device__ __forceinline__ u64 find(const W* hist, G target_of) {
    constexpr int PER = kBins / TH;
    const int tid = threadIdx.x, w = tid >> 6;
    u64 own[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += own[i] = hist[PER * tid + i];
    u64 up = wave_scan(sum);
    if ((tid & 63) == 63) lds.wave[w] = up;
    __syncthreads();
    up -= sum;
    u64 all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < w) up += lds.wave[i];
      all += lds.wave[i];
    }
    const u64 target = target_of(all);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (up < target && target <= up + own[i]) lds.bin = PER * tid + i, lds.before = up, lds.upto = up + own[i];
      up += own[i];
    }
    __syncthreads();
    return target;
  }
  // The tokens of least <= logit < end (of all from least on where end is −∞) in the list: their number,
  // of which the list holds the first kList.
  __device__ __forceinline__ int gather(float least, float end) {
    constexpr int AT_ONCE = 8;
    if (infinite) {  // logits as they lie in memory, of which only +∞ counts
      end = (least <= 0.f && (0.f < end || end == -INFINITY)) ? -INFINITY : NAN;
      least = INFINITY;
    }
    __syncthreads();
    if (threadIdx.x == 0) lds.count = 0;
    __syncthreads();
    for (int c = 0; c < n_chunks; c += AT_ONCE) {
      floatx4 v[AT_ONCE];
      raw(c, v);
      u64 hits = 0;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        uint32 four = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) four |= (uint32)(v[i][e] >= least && (v[i][e] < end || end == -INFINITY)) << e;
        hits |= (u64)four << (4 * i);
      }
      for (; hits; hits &= hits - 1) {
        const int bit = __builtin_ctzll(hits), at = 4 * ((c + (bit >> 2)) * TH + (int)threadIdx.x) + (bit & 3);
        const int n = atomicAdd(&lds.count, 1);
        if (n < kList) lds.list[n].i = at;
      }
    }
    __syncthreads();
    for (int n = threadIdx.x; n < min(lds.count, kList); n += TH) {
      const int at = lds.list[n].i;
      const float v = infinite ? 0.f : x[at];
      lds.list[n] = Entry{v, at, weight(v)};
    }
    __syncthreads();
    return lds.count;
  }

  // Of the order of falling logits, rising indexes: the place at which the sum of weights f(index, logit)
  // reaches target(the sum of all), as its logit and index: 1.  There is none: 0.  f is the same for equal
  // logits, but for a last part of them in the order that has none.
  // few > 0: where that place's range and all above it hold no more than `few` tokens of a weight, these go
  // into the list, lds.count of them: 2.
  template <class F, class G>
  __device__ __forceinline__ int reach(F f, G target_of, int few, float& at_x, int& at_i) {
    using W = decltype(f(0, 0.f));
    W* const hist = reinterpret_cast<W*>(lds.hist);
    // the first ranges end where weights do; all below them share the last one
    Ranges ranges = first_ranges(m, T);
    float lo = -INFINITY;
    u64 target = 0;
    for (bool first = true;; first = false) {
      auto bin_of = [&](float v) { return ranges.of(v); };
      auto in = [&](float v) { return v > -INFINITY && v >= lo && (double)v <= ranges.hi; };
      clear();
      each(0, n_chunks, [&](int, int i, floatx4 v) {
        one_by_one(v, i, [&](int at, float y) {
          if (!in(y)) return;
          const W x = f(at, y);
          if (x) atomicAdd(&hist[bin_of(y)], x);
        });
      });
      __syncthreads();
      target = find(hist, [&](u64 all) { return first ? target_of(all) : target; });
      const int bin = lds.bin;
      if (bin < 0) return 0;
      target -= lds.before;
      if (first && lds.upto <= (u64)few) {  // (weights of one each: f counts)
        each(0, n_chunks, [&](int, int i, floatx4 v) {
          one_by_one(v, i, [&](int at, float y) {
            if (in(y) && bin_of(y) <= bin) lds.list[atomicAdd(&lds.count, 1)] = Entry{y, at, 0};
          });
        });
        __syncthreads();
        return 2;
      }
      float most = -INFINITY, fewest = INFINITY;
      each(0, n_chunks, [&](int, int i, floatx4 v) {
        one_by_one(v, i, [&](int at, float y) {
          if (!in(y) || bin_of(y) != bin) return;
          most = fmaxf(most, y);
          fewest = fminf(fewest, y);
          const int n = atomicAdd(&lds.count, 1);
          if (n < kList) lds.list[n] = Entry{y, at, f(at, y)};
        });
      });
      __syncthreads();
      const int n = lds.count;
      if (n <= kList) {
        const Entry at = reach_in_list(n, target, [](const Entry& e) { return e.w; }, ranges, bin);
        at_x = at.x;
        at_i = at.i;
        return 1;
      }
      const float top = block_max(most);
      lo = -block_max(-fewest);
      if (lo == top) {  // one value: its tokens in the order of their indexes
        const float v = lo;
        const u64 one = f(0, v);
        u64 none;
        at_x = v;
        at_i = pick([v](int, float y) { return (u64)(y == v); }, [&](u64) { return (target + one - 1) / one - 1; }, none);
        return 1;
      }
      // (in 64 bits, where no difference of two logits is lost: lo and hi never share a range)
      ranges = {top, kBins / ((double)top - (double)lo)};
    }
  }

  // The choice among the n <= TH / 4 tokens in the list, the first k of which count.  Four threads have a token.
  __device__ __forceinline__ void choose_few(int r, int n, int k, float p, float least) {
    const int e = threadIdx.x >> 2, part = threadIdx.x & 3;
    const bool on = e < n;
    Entry own{-INFINITY, 0x7fffffff, 0};
    if (on) own = lds.list[e];
    uint32 rank = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 4) rank += before(lds.list[j].x, lds.list[j].i, own.x, own.i);
    rank = (uint32)quad_sum(rank);
    own.w = on && (int)rank < k ? weight(own.x) : 0;
    if (on && part == 0) lds.list[e].w = own.w;
    __syncthreads();
    u64 sum = 0, ahead = 0;
    if (p < 1.f) {
#pragma unroll 4
      for (int j = part; j < n; j += 4) {
        const Entry o = lds.list[j];
        sum += o.w;
        ahead += before(o.x, o.i, own.x, own.i) ? o.w : 0;
      }
      sum = quad_sum(sum);
      ahead = quad_sum(ahead);
      if ((double)ahead >= (double)p * (double)sum && ahead > 0) own.w = 0;
    }
    if (own.x < least) own.w = 0;
    __syncthreads();
    if (on && part == 0) lds.list[e].w = own.w;
    __syncthreads();
    sum = ahead = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 4) {
      const Entry o = lds.list[j];
      sum += o.w;
      ahead += o.i < own.i ? o.w : 0;
    }
    sum = quad_sum(sum);
    ahead = quad_sum(ahead);
    const u64 at = place(r, sum);
    if (on && part == 0 && ahead <= at && at < ahead + own.w) result(r, own.i, own.x, sum);
  }

  // u times the sum, rounded down, below it.
  __device__ __forceinline__ u64 place(int r, u64 total) const {
    const float u = a.u[r];
    const double want = (double)(u > 0.f ? u : 0.f) * (double)total;
    const u64 at = want < (double)total ? (u64)want : total - 1;
    return at < total ? at : total - 1;
  }
  __device__ __forceinline__ void result(int r, int token, float v, u64 total) const {
    a.tokens[r] = token;
    if (a.logprob) {
      const double y = v == m ? 0.0 : ((double)v - (double)m) * inv_t;
      a.logprob[r] = (float)(y - log(ldexp((double)total, -a.frac)));
    }
  }
};

// The row's logits from cut_x on, at cut_x those of indexes up to cut_i.
struct Cut {
  float x;
  int i;
  __device__ __forceinline__ bool keeps(float v, int at) const { return v > x || (v == x && at <= i); }
  // Of all logits from v on as well.
  __device__ __forceinline__ bool above(float v) {
    if (!(x < v)) return false;
    x = v;
    i = 0x7fffffff;
    return true;
  }
};

// Borders and choice by passes over the whole row.
template <int TH, int ROW>
__device__ __forceinline__ void choose(Row<TH, ROW>& row, const Filters& f, int r) {
  Cut cut{-INFINITY, 0x7fffffff};
  if (f.k > 0 &&
      row.reach([](int, float) { return 1u; }, [&](u64) { return (u64)f.k; }, TH / 4, cut.x, cut.i) == 2) {
    row.choose_few(r, row.lds.count, f.k, f.p, f.least(row.m));
    return;
  }
  if (f.p < 1.f) {
    const Cut by_k = cut;
    auto all = [&](int i, float v) { return by_k.keeps(v, i) ? row.weight(v) : (u64)0; };
    row.reach(all, [&](u64 mass) { return p_target(f.p, mass); }, 0, cut.x, cut.i);
  }
  cut.above(f.least(row.m));
  auto kept = [&](int i, float v) { return cut.keeps(v, i) ? row.weight(v) : (u64)0; };
  u64 total;
  const int token = row.pick(kept, [&](u64 sum) { return row.place(r, sum); }, total);
  if (threadIdx.x == 0) row.result(r, token, row.infinite ? 0.f : row.x[token], total);
}

// The same out of line, for rows that hardly ever come.
// They get a row of their own, for one whose address another function gets lies in memory wherever it is used.
template <int TH, int ROW>
__device__ __attribute__((noinline)) void choose_apart(const SampleArgs& a, SampleLds& lds, int r, float most, float T) {
  Row<TH, ROW> row(a, lds, nullptr, r);
  row.take(most, T);
  choose(row, Filters(a, r), r);
}

// A row without anything to choose from; nor with a choice to make: its first largest logit.
__device__ __forceinline__ void certain(const SampleArgs& a, int r, int token, float logprob) {
  a.tokens[r] = token;
  if (a.logprob) a.logprob[r] = logprob;
}

// ROW: 4-logit pieces of a row in LDS.
template <int TH, int ROW>
__global__ void __launch_bounds__(TH) sample_kernel(SampleArgs a) {
  __shared__ SampleLds lds;
  __shared__ floatx4 held[ROW];
  const int r = blockIdx.x, tid = threadIdx.x;
  Row<TH, ROW> row(a, lds, held, r);
  const Filters f(a, r);
  float most = -INFINITY;
  constexpr int AT_ONCE = ROW / TH < 4 ? ROW / TH : 4;
  for (int c = 0; c < row.n_chunks; c += AT_ONCE) {
    floatx4 v[AT_ONCE];
    row.raw(c, v);
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      v[i] = row.clean(v[i]);
      held[(c + i) * TH + tid] = v[i];
      most = fmaxf(fmaxf(most, fmaxf(v[i][0], v[i][1])), fmaxf(v[i][2], v[i][3]));
    }
  }
  row.take(row.block_max(most), f.T);
  if (row.m == -INFINITY) {
    if (tid == 0) certain(a, r, 0, -INFINITY);
    return;
  }
  if (row.infinite)
    for (int c = 0; c < row.n_chunks; ++c) held[c * TH + tid] = row.ordinary(held[c * TH + tid]);
  if (f.greedy()) {
    const int token = row.first_of(row.m, 0, row.n_chunks);
    if (tid == 0) certain(a, r, token, 0.f);
    return;
  }
  choose(row, f, r);
}

// ---------------------------------------------------------------- rows that several blocks share

// Three launches: the segments' largest logits; with the row's largest their histograms of weights (and of counts
// for top_k) and the weight of what min_p keeps; a block a row, which adds these up, collects the tokens of the one
// or two ranges that hold its borders from the row, and goes through the weights of the part of a segment that the
// random number falls into (of the whole segment where a list decides which are kept).  64 rows of 131072: 7, 17 and
// 23 us where min_p's border is the higher one, 43 for the last where top_p's tokens are collected; reading the
// logits once takes 7.  The second is bound by its arithmetic in 64 bits, the last by how long one block takes.

__global__ void __launch_bounds__(512) sample_max_kernel(SampleArgs a) {
  __shared__ SampleLds lds;
  const int r = blockIdx.x / a.segments, g = blockIdx.x % a.segments;
  Row<512, 0> row(a, lds, nullptr, r);
  floatx4 v[kSegment / 2048];
  float most = -INFINITY;
  row.raw(g * (kSegment / 2048), v);
#pragma unroll
  for (int c = 0; c < kSegment / 2048; ++c) v[c] = row.clean(v[c]);
#pragma unroll
  for (int c = 0; c < kSegment / 2048; ++c) most = fmaxf(fmaxf(most, fmaxf(v[c][0], v[c][1])), fmaxf(v[c][2], v[c][3]));
  most = row.block_max(most);
  if (threadIdx.x == 0) a.seg_max[blockIdx.x] = most;
}

__device__ __forceinline__ float row_max(const SampleArgs& a, int r) {
  const int lane = threadIdx.x & 63;
  return aurlanes::group_reduce<1, 64, true>(lane < a.segments ? a.seg_max[(size_t)r * a.segments + lane] : -INFINITY);
}

__global__ void __launch_bounds__(512) sample_histogram_kernel(SampleArgs a) {
  __shared__ SampleLds lds;
  __shared__ uint32 counts[kBins];
  const int r = blockIdx.x / a.segments, g = blockIdx.x % a.segments, tid = threadIdx.x;
  Row<512, 0> row(a, lds, nullptr, r);
  // a wave has 2048 tokens that follow each other, so its sum is one of a part of the row
  constexpr int N = kSegment / 2048;
  const int first = g * kSegment + (tid >> 6) * 2048 + 4 * (tid & 63);
  floatx4 v[N];
  if ((g + 1) * kSegment <= a.vocab) {
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = *reinterpret_cast<const floatx4_any*>(row.x + first + 256 * c);
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[c][e] = first + 256 * c + e < a.vocab ? row.x[first + 256 * c + e] : -INFINITY;
  }
  const Filters f(a, r);
  row.take(row_max(a, r), f.T);
  if (row.m == -INFINITY || f.greedy()) return;
  const bool borders = f.k > 0 || f.p < 1.f;
  if (borders)
    for (int i = tid; i < kBins; i += 512) lds.hist[i] = counts[i] = 0;
  __syncthreads();
  const Ranges ranges = first_ranges(row.m, f.T);
  const float least = f.least(row.m);
  u64 sum = 0;
  Series series;
  series.keep();
#pragma unroll 1
  for (int c = 0; c < N; ++c) {
    const floatx4 x = row.clean(v[0]);
#pragma unroll
    for (int i = 0; i + 1 < N; ++i) v[i] = v[i + 1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!(x[e] > -INFINITY)) continue;
      const u64 w = weight_of(x[e], row.m, row.scale, a.frac, series);
      if (x[e] >= least) sum += w;
      if (!borders) continue;
      const int bin = ranges.of(x[e]);
      if (f.k > 0) atomicAdd(&counts[bin], 1u);
      if (w) atomicAdd(&lds.hist[bin], w);
    }
  }
  sum = wave_sum(sum);
  if ((tid & 63) == 0) lds.wave[tid >> 6] = sum;
  __syncthreads();
  if (borders)
    for (int i = tid; i < kBins; i += 512) {
      a.mass[(size_t)blockIdx.x * kBins + i] = lds.hist[i];
      if (f.k > 0) a.count[(size_t)blockIdx.x * kBins + i] = counts[i];
    }
  if (tid < kParts) a.seg_mass[(size_t)blockIdx.x * kParts + tid] = lds.wave[2 * tid] + lds.wave[2 * tid + 1];
}

__global__ void __launch_bounds__(1024) sample_finish_kernel(SampleArgs a) {
  constexpr int TH = 1024, CHUNKS = kSegment / (4 * TH);
  static_assert(CHUNKS == kParts, "a part is a chunk");
  __shared__ SampleLds lds;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, G = a.segments;
  // this thread's range over all segments (what lies there where no histogram was made is not used)
  const u64* const mass = a.mass + (size_t)r * G * kBins;
  const uint32* const count = a.count + (size_t)r * G * kBins;
  u64 own_count = 0, own_mass = 0;
#pragma unroll 8
  for (int g = 0; g < G; ++g) own_mass += mass[(size_t)g * kBins + tid];
  Row<TH, 0> row(a, lds, nullptr, r);
  const Filters f(a, r);
  if (f.k > 0) {
#pragma unroll 8
    for (int g = 0; g < G; ++g) own_count += count[(size_t)g * kBins + tid];
  }
  row.take(row_max(a, r), f.T);
  if (row.m == -INFINITY) {
    if (tid == 0) certain(a, r, 0, -INFINITY);
    return;
  }
  if (f.greedy()) {
    const float top = row.infinite ? INFINITY : row.m;  // as the segments have it
    const int g = __builtin_ctzll(__ballot(lane < G && a.seg_max[(size_t)r * G + lane] == top));
    const int token = row.first_of(row.m, g * CHUNKS, min((g + 1) * CHUNKS, row.n_chunks));
    if (tid == 0) certain(a, r, token, 0.f);
    return;
  }
  Cut cut{-INFINITY, 0x7fffffff};
  const float least = f.least(row.m);
  int listed = -1, n = 0;  // the range whose tokens are in the list
  if (f.k > 0 || f.p < 1.f) {
    const Ranges ranges = first_ranges(row.m, f.T);
    const int least_bin = least > kLeastLogit ? ranges.of(least) : kBins;
    u64 kept_mass = 0;  // of the first top_k
    bool crowded = false, below = false;  // more than the list holds: by passes over the row then
    // The range where `own` reaches the target, and its tokens in the list; what is left of the target there.  A
    // border that only matters where it lies above min_p's is not looked for in a range below that one.
    auto search = [&](u64 own, bool last, auto target_of) {
      row.clear();
      lds.hist[tid] = own;
      __syncthreads();
      const u64 target = row.find(lds.hist, target_of);
      const int bin = lds.bin;
      const u64 rest = target - (bin < 0 ? 0 : lds.before);
      below = last && bin > least_bin;
      if (bin >= 0 && bin != listed && !below) {
        n = row.gather(ranges.edge(bin), bin > 0 ? ranges.edge(bin - 1) : -INFINITY);
        listed = bin;
        crowded = n > kList;
      }
      return rest;
    };
    if (f.k > 0) {
      const u64 rest = search(own_count, f.p == 1.f, [&](u64) { return (u64)f.k; });
      if (listed >= 0 && !crowded) {
        const Entry at = row.reach_in_list(n, rest, [](const Entry&) { return (u64)1; }, ranges, listed);
        cut = Cut{at.x, at.i};
        if (f.p < 1.f) {  // the weight of all kept
          __syncthreads();
          if (tid == 0) lds.upto = 0;
          __syncthreads();
          u64 sum = tid < listed ? own_mass : 0;
          for (int i = tid; i < n; i += TH) sum += cut.keeps(lds.list[i].x, lds.list[i].i) ? lds.list[i].w : 0;
          sum = wave_sum(sum);
          if (lane == 0) atomicAdd(&lds.upto, sum);
          __syncthreads();
          kept_mass = lds.upto;
        }
      }
    }
    if (f.p < 1.f && !crowded) {
      const bool by_k = listed >= 0;
      const u64 rest = search(own_mass, true, [&](u64 all) { return p_target(f.p, by_k ? kept_mass : all); });
      if (!crowded && !below) {
        const Entry at = row.reach_in_list(n, rest, [](const Entry& e) { return e.w; }, ranges, listed);
        cut = Cut{at.x, at.i};
      }
    }
    if (crowded) {
      choose_apart<TH, 0>(a, lds, r, row.infinite ? INFINITY : row.m, f.T);
      return;
    }
    if (below) listed = -1;
  }
  // The segments' kept weights: above min_p's border, or of the ranges above the listed one and of the tokens in it.
  if (cut.above(least)) listed = -1;
  __syncthreads();
  if (listed < 0) {
    if (tid < G) {
      const u64* const m = a.seg_mass + ((size_t)r * G + tid) * kParts;
      lds.super[tid] = m[0] + m[1] + m[2] + m[3];
    }
    __syncthreads();
  } else {
    for (int g = w; g < G; g += TH / 64) {
      u64 sum = 0;
#pragma unroll
      for (int i = 0; i < kBins / 64; ++i) {
        const u64 x = mass[(size_t)g * kBins + 64 * i + lane];
        sum += 64 * i + lane < listed ? x : 0;
      }
      sum = wave_sum(sum);
      if (lane == 0) lds.super[g] = sum;
    }
    __syncthreads();
    for (int i = tid; i < n; i += TH)
      if (cut.keeps(lds.list[i].x, lds.list[i].i)) atomicAdd(&lds.super[lds.list[i].i / kSegment], lds.list[i].w);
    __syncthreads();
  }
  auto kept = [&](int i, float v) { return cut.keeps(v, i) ? row.weight(v) : (u64)0; };
  const u64 total = row.sum_of(lds.super, G);
  u64 at = row.place(r, total);
  const int g = row.locate(lds.super, G, at);
  int c0 = g * CHUNKS, c1 = min(c0 + CHUNKS, row.n_chunks);
  if (listed < 0) {
    if (tid < kParts) lds.wave[tid] = a.seg_mass[((size_t)r * G + g) * kParts + tid];
    __syncthreads();
    c0 += row.locate(lds.wave, kParts, at);
    c1 = c0 + 1;
  }
  __syncthreads();
  row.sum_waves(c0, c1, kept);
  const int token = row.pick_in(c0, c1, at, kept);
  if (tid == 0) row.result(r, token, row.infinite ? 0.f : row.x[token], total);
}

// A row that fits is chosen from by one block out of LDS: at 32768 tokens that takes 16 us from all of them, 37 with
// top_p and 17 with top_k = 50 and top_p, three launches on segments of 40000 35, 52 and 58.
int segments_of(uint32_t vocab) { return vocab > (uint32_t)kStaged ? (int)((vocab + kSegment - 1) / kSegment) : 0; }

}  // namespace

extern "C" size_t aur_sample_ws_bytes(uint32_t b, uint32_t vocab) {
  if (vocab > (uint32_t)kMaxVocab || b > 0x000fffffu) return 0;
  const size_t n = (size_t)b * segments_of(vocab);
  return (n * (kBins * 12 + 8 * kParts + 4) + 15) / 16 * 16;
}

extern "C" int aur_sample(aur_ctx* ctx, const float* logits, uint32_t ld, const float* u, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
                          float* logprob, void* scratch, size_t scratch_bytes, uint32_t b, uint32_t vocab) {
  AUR_CHECK_CTX(ctx);
  const char* who = "aur_sample";
  if (vocab == 0 || ld < vocab)
    return aur::set_error(ctx, AUR_EINVAL, "%s: ld=%u of vocab=%u", who, ld, vocab);
  if (vocab > kMaxVocab || b > 0x000fffffu || ld > 0x7fffffffu)
    return aur::set_error(ctx, AUR_ELIMIT, "%s: b=%u vocab=%u (up to %d) ld=%u", who, b, vocab, kMaxVocab, ld);
  if (b == 0) return 0;
  if (!logits || !u || !tokens) return aur::set_error(ctx, AUR_EINVAL, "%s: null logits, u or tokens", who);
  int bits = 0;
  while ((1u << bits) < vocab) ++bits;
  SampleArgs a{logits, u, temperature, top_p, min_p, top_k, tokens, logprob, (int)vocab, (int)ld,
               63 - bits < 50 ? 63 - bits : 50};
  a.segments = segments_of(vocab);
  if (a.segments) {
    if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) || scratch_bytes < aur_sample_ws_bytes(b, vocab))
      return aur::set_error(ctx, AUR_EINVAL, "%s: scratch of %zu bytes (16-byte aligned), %zu needed", who,
                            scratch ? scratch_bytes : (size_t)0, aur_sample_ws_bytes(b, vocab));
    const size_t n = (size_t)b * a.segments;
    a.mass = static_cast<u64*>(scratch);
    a.seg_mass = a.mass + n * kBins;
    a.count = reinterpret_cast<uint32*>(a.seg_mass + n * kParts);
    a.seg_max = reinterpret_cast<float*>(a.count + n * kBins);
    hipLaunchKernelGGL(sample_max_kernel, dim3((unsigned)n), dim3(512), 0, ctx->stream, a);
    AUR_LAUNCH_CHECK(ctx, "sample_max_kernel");
    hipLaunchKernelGGL(sample_histogram_kernel, dim3((unsigned)n), dim3(512), 0, ctx->stream, a);
    AUR_LAUNCH_CHECK(ctx, "sample_histogram_kernel");
    hipLaunchKernelGGL(sample_finish_kernel, dim3(b), dim3(1024), 0, ctx->stream, a);
    AUR_LAUNCH_CHECK(ctx, "sample_finish_kernel");
    return 0;
  }
  // More threads pass over a long row sooner, fewer meet each other sooner at its barriers (top_p 0.95 on 32 rows,
  // us by 256, 512 and 1024 threads: 8.3, 9.0 and 10.0 at 1000 tokens, 14.6, 11.8 and 12.1 at 4096, 22.7, 16.6 and
  // 15.8 at 8192; drawn from all tokens 9.2, 7.9 and 7.8 there).
  auto* kernel = vocab <= 1024   ? sample_kernel<256, 256>
                 : vocab <= 8192 ? sample_kernel<512, 2048>
                                 : sample_kernel<1024, kStaged / 4>;
  const dim3 threads(vocab <= 1024 ? 256 : vocab <= 8192 ? 512 : 1024);
  hipLaunchKernelGGL(kernel, dim3(b), threads, 0, ctx->stream, a);
  AUR_LAUNCH_CHECK(ctx, "sample_kernel");
  return 0;
}
