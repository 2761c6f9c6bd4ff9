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

#include <cmath>

namespace {

typedef unsigned long long u64;
typedef unsigned uint32;

struct SampleArgs {
  const float *logits, *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* tokens;
  float* logprob;
  int vocab, ld, frac;  // weights in units of 2^-frac
  bool aligned;         // rows of whole 16-byte pieces
};

constexpr int kBins = 1024, kList = 1024;
constexpr int kSuper = 8;          // chunks whose weights are added up together
constexpr int kMaxVocab = 1 << 20;
constexpr int kStaged = 32768;     // logits of a row in LDS

struct Entry {
  float x;
  int i;
  u64 w;
};

struct SampleLds {
  u64 hist[kBins];
  __attribute__((aligned(16))) Entry list[kList];
  u64 wave[kSuper * 16];
  u64 super[kMaxVocab / (4 * 1024 * kSuper) + 1];
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
  bool infinite;  // the largest logit is +∞: such ones count as 0, all others as −∞

  __device__ __forceinline__ floatx4 ordinary(floatx4 v) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] == INFINITY ? 0.f : -INFINITY;
    return v;
  }
  // A logit that is NaN counts as −∞, and so does what lies behind the row.
  __device__ __forceinline__ floatx4 load(int c) const {
    const int i = 4 * (c * TH + threadIdx.x);
    floatx4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (a.aligned && i + 3 < a.vocab) {
      v = *reinterpret_cast<const floatx4*>(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < a.vocab) v[e] = x[i + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] == v[e] ? v[e] : -INFINITY;
    return infinite ? ordinary(v) : v;
  }
  // f(chunk, index of the first, four logits) for the chunks from c0 up to c1.
  template <class F>
  __device__ __forceinline__ void each(int c0, int c1, F f) const {
    for (int c = c0; c < c1; ++c) f(c, 4 * (c * TH + (int)threadIdx.x), ROW ? held[c * TH + threadIdx.x] : load(c));
  }

  // The weight of logit v in units of 2^-frac, to the nearest.
  __device__ __forceinline__ u64 weight(float v) const {
    const double y = fmax(((double)v - (double)m) * scale, -2000.0);
    const double n = __builtin_rint(y), r = (y - n) * 0.6931471805599453;
    double p = 1.0 / 39916800.0;
#define AUR_TERM(k) p = __builtin_fma(p, r, 1.0 / k)
    AUR_TERM(3628800.0);
    AUR_TERM(362880.0);
    AUR_TERM(40320.0);
    AUR_TERM(5040.0);
    AUR_TERM(720.0);
    AUR_TERM(120.0);
    AUR_TERM(24.0);
    AUR_TERM(6.0);
    AUR_TERM(2.0);
    AUR_TERM(1.0);
    AUR_TERM(1.0);
#undef AUR_TERM
    p = __builtin_rint(ldexp(p, (int)n + a.frac));  // up to 2^50
    const double hi = __builtin_floor(p * 0x1p-32);
    return (u64)(uint32)hi << 32 | (uint32)__builtin_fma(hi, -0x1p32, p);
  }

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
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += f(i + e, v[e]);
      sum = wave_sum(sum);
      if ((threadIdx.x & 63) == 0) lds.wave[(c - c0) * NW + (threadIdx.x >> 6)] = sum;
    });
    __syncthreads();
  }
  // The least index at which the sum of the weights f(index, logit) up to it exceeds place(their sum).
  template <class F, class G>
  __device__ __forceinline__ int pick(F f, G place, u64& total) {
    const int w = threadIdx.x >> 6, n = (n_chunks + kSuper - 1) / kSuper;
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
        each(s * kSuper, min((s + 1) * kSuper, n_chunks), [&](int, int i, floatx4 v) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += f(i + e, v[e]);
        });
        sum = wave_sum(sum);
        if ((threadIdx.x & 63) == 0) atomicAdd(&lds.super[s], sum);
      }
      __syncthreads();
      total = sum_of(lds.super, n);
      r = place(total);
      c0 = locate(lds.super, n, r) * kSuper;
      sum_waves(c0, min(c0 + kSuper, n_chunks), f);
    }
    const int at = locate(lds.wave, min(kSuper, n_chunks - c0) * NW, r);
    if (w == at % NW)
      each(c0 + at / NW, c0 + at / NW + 1, [&](int, int i, floatx4 v) {
        u64 t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = f(i + e, v[e]);
        u64 up = wave_scan(t[0] + t[1] + t[2] + t[3]) - (t[0] + t[1] + t[2] + t[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (up <= r && r < up + t[e]) lds.token = i + e;
          up += t[e];
        }
      });
    __syncthreads();
    return lds.token;
  }

  // Of the order of falling logits, rising indexes: the place at which the sum of weights f(index, logit)
  // reaches target(the sum of all), as its logit and index: 1.  There is none: 0.  f is the same for equal
  // logits, but for a last part of them in the order that has none.
  // few > 0: where that place's range and all above it hold no more than `few` tokens of a weight, these go
  // into the list, lds.count of them: 2.
  template <class F, class G>
  __device__ __forceinline__ int reach(F f, G target_of, int few, float& at_x, int& at_i) {
    using W = decltype(f(0, 0.f));
    constexpr int PER = kBins / TH;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    W* const hist = reinterpret_cast<W*>(lds.hist);
    // the first ranges end where weights do; all below them share the last one
    double hi = m, inv = kBins / (32.0 * (double)T);
    float lo = -INFINITY;
    u64 target = 0;
    for (bool first = true;; first = false) {
      auto bin_of = [&](float v) { return (int)fmin((hi - (double)v) * inv, kBins - 1.0); };
      auto in = [&](float v) { return v > -INFINITY && v >= lo && (double)v <= hi; };
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i) hist[tid + TH * i] = 0;
      if (tid == 0) lds.bin = -1, lds.count = 0;
      __syncthreads();
      each(0, n_chunks, [&](int, int i, floatx4 v) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in(v[e])) {
            const W x = f(i + e, v[e]);
            if (x) atomicAdd(&hist[bin_of(v[e])], x);
          }
      });
      __syncthreads();
      u64 own[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += own[i] = hist[PER * tid + i];
      u64 up = wave_scan(sum);
      if (lane == 63) lds.wave[w] = up;
      __syncthreads();
      up -= sum;
      u64 all = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        if (i < w) up += lds.wave[i];
        all += lds.wave[i];
      }
      if (first) target = target_of(all);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (up < target && target <= up + own[i]) lds.bin = PER * tid + i, lds.before = up, lds.upto = up + own[i];
        up += own[i];
      }
      __syncthreads();
      const int bin = lds.bin;
      if (bin < 0) return 0;
      target -= lds.before;
      if (first && lds.upto <= (u64)few) {  // (weights of one each: f counts)
        each(0, n_chunks, [&](int, int i, floatx4 v) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (in(v[e]) && bin_of(v[e]) <= bin) lds.list[atomicAdd(&lds.count, 1)] = Entry{v[e], i + e, 0};
        });
        __syncthreads();
        return 2;
      }
      float most = -INFINITY, fewest = INFINITY;
      each(0, n_chunks, [&](int, int i, floatx4 v) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in(v[e]) && bin_of(v[e]) == bin) {
            most = fmaxf(most, v[e]);
            fewest = fminf(fewest, v[e]);
            const int n = atomicAdd(&lds.count, 1);
            if (n < kList) lds.list[n] = Entry{v[e], i + e, f(i + e, v[e])};
          }
      });
      __syncthreads();
      const int n = lds.count;
      if (n <= kList) {
        for (int i = tid; i < n; i += TH) {
          const Entry own_e = lds.list[i];
          u64 sum_before = 0;
#pragma unroll 4
          for (int j = 0; j < n; ++j) {
            const Entry o = lds.list[j];
            sum_before += before(o.x, o.i, own_e.x, own_e.i) ? o.w : 0;
          }
          if (sum_before < target && target <= sum_before + own_e.w) lds.best = i;
        }
        __syncthreads();
        at_x = lds.list[lds.best].x;
        at_i = lds.list[lds.best].i;
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
      hi = top;
      inv = kBins / (hi - (double)lo);
    }
  }

  // The choice among the n <= TH / 4 tokens in the list, the first k of which count.  Four threads have a token.
  __device__ __forceinline__ void choose_few(int r, int n, int k, float p, double floor_y) {
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
    if (own.x != m && !(((double)own.x - (double)m) * inv_t >= floor_y)) own.w = 0;
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

// ROW: 4-logit pieces of a row in LDS.
template <int TH, int ROW>
__global__ void __launch_bounds__(TH) sample_kernel(SampleArgs a) {
  __shared__ SampleLds lds;
  __shared__ floatx4 held[ROW ? ROW : 1];
  const int r = blockIdx.x, tid = threadIdx.x;
  Row<TH, ROW> row{a, lds, held, a.logits + (size_t)r * a.ld, (a.vocab + 4 * TH - 1) / (4 * TH)};
  const float T = a.temperature ? a.temperature[r] : 1.f, p = a.top_p ? a.top_p[r] : 1.f;
  const float least_p = a.min_p ? a.min_p[r] : 0.f;
  int k = a.top_k ? a.top_k[r] : 0;
  if (k >= a.vocab || k < 0) k = 0;
  row.infinite = false;
  float most = -INFINITY;
  for (int c = 0; c < row.n_chunks; ++c) {
    const floatx4 v = row.load(c);
    if (ROW) held[c * TH + tid] = v;
    most = fmaxf(fmaxf(most, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));
  }
  row.m = row.block_max(most);
  if (row.m == -INFINITY) {  // nothing to choose from
    if (tid == 0) {
      a.tokens[r] = 0;
      if (a.logprob) a.logprob[r] = -INFINITY;
    }
    return;
  }
  row.infinite = row.m == INFINITY;
  if (row.infinite) {
    row.m = 0.f;
    if (ROW)
      for (int c = 0; c < row.n_chunks; ++c) held[c * TH + tid] = row.ordinary(held[c * TH + tid]);
  }
  if (!(T > 0.f) || k == 1 || p <= 0.f) {  // greedy: the first of the largest
    int token = 0x7fffffff;
    const float m = row.m;
    row.each(0, row.n_chunks, [&](int, int i, floatx4 v) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[e] == m) token = min(token, i + e);
    });
    if (tid == 0) lds.token = 0x7fffffff;
    __syncthreads();
    if (token != 0x7fffffff) atomicMin(&lds.token, token);
    __syncthreads();
    if (tid == 0) {
      a.tokens[r] = lds.token;
      if (a.logprob) a.logprob[r] = 0.f;
    }
    return;
  }
  row.T = T;
  row.inv_t = 1.0 / (double)T;
  row.scale = 1.4426950408889634 / (double)T;
  const float m = row.m;
  const double floor_y = least_p > 0.f ? log((double)fminf(least_p, 1.f)) : -INFINITY;

  // The kept tokens: logits above cut_x, and at cut_x indexes up to cut_i.
  float cut_x = -INFINITY;
  int cut_i = 0x7fffffff;
  if (k > 0 &&
      row.reach([](int, float) { return 1u; }, [k](u64) { return (u64)k; }, TH / 4, cut_x, cut_i) == 2) {
    row.choose_few(r, lds.count, k, p, floor_y);
    return;
  }
  if (p < 1.f) {
    const float kx = cut_x;
    const int ki = cut_i;
    auto all = [&](int i, float v) { return v > kx || (v == kx && i <= ki) ? row.weight(v) : (u64)0; };
    row.reach(all, [p](u64 mass) { return (u64)fmax(ceil((double)p * (double)mass), 1.0); }, 0, cut_x, cut_i);
  }
  auto kept = [&](int i, float v) {
    const bool in = (v > cut_x || (v == cut_x && i <= cut_i)) && (v == m || ((double)v - (double)m) * row.inv_t >= floor_y);
    return in ? row.weight(v) : (u64)0;
  };
  u64 total;
  const int token = row.pick(kept, [&](u64 sum) { return row.place(r, sum); }, total);
  if (tid == 0) row.result(r, token, row.infinite ? 0.f : row.x[token], total);
}

}  // namespace

extern "C" int aur_sample(aur_ctx* ctx, const float* logits, uint32_t ld, const float* u, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
                          float* logprob, uint32_t b, uint32_t vocab) {
  AUR_CHECK_CTX(ctx);
  const char* who = "aur_sample";
  if (vocab == 0 || ld < vocab)
    return aur::set_error(ctx, AUR_EINVAL, "%s: ld=%u of vocab=%u", who, ld, vocab);
  if (vocab > kMaxVocab || b > 0x00ffffffu || ld > 0x7fffffffu)
    return aur::set_error(ctx, AUR_ELIMIT, "%s: b=%u vocab=%u (up to %d) ld=%u", who, b, vocab, kMaxVocab, ld);
  if (b == 0) return 0;
  if (!logits || !u || !tokens) return aur::set_error(ctx, AUR_EINVAL, "%s: null logits, u or tokens", who);
  int bits = 0;
  while ((1u << bits) < vocab) ++bits;
  SampleArgs a{logits, u, temperature, top_p, min_p, top_k, tokens, logprob, (int)vocab, (int)ld,
               63 - bits < 50 ? 63 - bits : 50, ld % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0};
  auto* kernel = vocab <= 256      ? sample_kernel<256, 256>
                 : vocab <= 8192    ? sample_kernel<512, 2048>
                 : vocab <= kStaged ? sample_kernel<1024, kStaged / 4>
                                    : sample_kernel<1024, 0>;
  const dim3 threads(vocab <= 256 ? 256 : vocab <= 8192 ? 512 : 1024);
  hipLaunchKernelGGL(kernel, dim3(b), threads, 0, ctx->stream, a);
  AUR_LAUNCH_CHECK(ctx, "sample_kernel");
  return 0;
}
