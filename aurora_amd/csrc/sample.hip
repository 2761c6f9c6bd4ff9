// The next token of each row of logits, from a random number that the caller gives.
//
// With m the row's largest logit, a token's weight is w = exp((x − m) / T).  In the order of
// falling logits, equal ones by rising index, the kept tokens are a first part of the row: the
// first top_k; of these the fewest whose weight reaches top_p of the first top_k's; of these
// the ones with w >= min_p; the first one always.  The token is the least index i at which the
// sum of the kept weights up to it, in the order of the indexes, exceeds u times their sum.
//
// Whether a token is kept, and which one is drawn, hangs on sums that pass a border, so these
// have to come out the same in any order: a weight is computed in 64 bits (2^y = 2^n·2^(i/64)·e^r
// with a table of 64 and five terms of e^r's series, |r| < 0.0055, to 2^-52) and held as a whole
// number of units of 2^-F, F = 63 − ⌈log2 vocab⌉ up to 50, so that a row's sum stays below 2^63.
// Whole numbers add up exactly, which lets threads and atomics add them as they come.
//
// The border of top_k or top_p is found by one histogram over 1024 equal ranges of logits (each
// range's count or weight), a scan over it, and the exact order among the tokens of the one range
// that holds the border.  Where more than 1024 tokens lie in it, it is cut into 1024 again; a
// range of one value alone is cut by index.
#include "common.hpp"

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
constexpr int kSuper = 8;                 // chunks whose weights are added up together
constexpr int kMaxVocab = 1 << 20;

struct SampleLds {
  u64 hist[kBins];
  u64 list_w[kList];
  float list_x[kList];
  int list_i[kList];
  double pow2[64];                        // 2^(i/64)
  u64 wave[kSuper * 16];
  u64 super[kMaxVocab / (4 * 1024 * kSuper) + 1];
  float red[2][16];
  u64 before, total;
  int bin, count, best, token;
};

__device__ __forceinline__ u64 shfl_up64(u64 x, int n) {
  const uint32 lo = __shfl_up((uint32)x, n, 64), hi = __shfl_up((uint32)(x >> 32), n, 64);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 shfl_xor64(u64 x, int n) {
  const uint32 lo = __shfl_xor((uint32)x, n, 64), hi = __shfl_xor((uint32)(x >> 32), n, 64);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_sum(u64 x) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x += shfl_xor64(x, o);
  return x;
}
__device__ __forceinline__ u64 wave_scan(u64 x) {  // of the lanes up to this one
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const u64 y = shfl_up64(x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// One row.  TH threads; the row lies in NCH chunks of 4 * TH logits in registers, or for NCH = 0 is read
// again in each pass.
template <int TH, int NCH>
struct Row {
  const SampleArgs& a;
  SampleLds& lds;
  const float* x;
  int n_chunks;
  floatx4 held[NCH ? NCH : 1];
  double scale;  // log2(e) / T
  float m;
  int frac;
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
  // f(index of the first, four logits) for every chunk from c0 on.
  template <class F>
  __device__ __forceinline__ void each(int c0, int c1, F f) {
    if constexpr (NCH > 0) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (c >= c0 && c < c1) f(c, 4 * (c * TH + (int)threadIdx.x), held[c]);
    } else {
      for (int c = c0; c < c1; ++c) f(c, 4 * (c * TH + (int)threadIdx.x), load(c));
    }
  }

  // The weight of logit v in units of 2^-frac, to the nearest.
  __device__ __forceinline__ u64 weight(float v) const {
    if (v == -INFINITY) return 0;
    if (v == m) return 1ull << frac;
    const double y = ((double)v - (double)m) * (scale * 64.0);  // in 64ths
    if (!(y > -64.0 * 64.0)) return 0;
    const double n = __builtin_rint(y), r = (y - n) * 0.010830424696249145;  // ln 2 / 64
    const int k = (int)n;
    double p = 1.0 / 120.0;
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    const u64 bits = (u64)__double_as_longlong(p * lds.pow2[k & 63]);
    const int shift = 52 - frac - (k >> 6) - ((int)(bits >> 52) - 1023);  // above 0: the weight is at most 1
    const u64 mant = (bits & 0xfffffffffffffull) | 0x10000000000000ull;
    return shift > 54 ? 0 : ((mant >> (shift - 1)) + 1) >> 1;
  }

  __device__ __forceinline__ float block_max(float v) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) v = fmaxf(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds.red[0][threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds.red[0][0];
#pragma unroll
    for (int w = 1; w < TH / 64; ++w) v = fmaxf(v, lds.red[0][w]);
    return v;
  }

  // Weights f(index, logit) added up by groups of kSuper chunks; their sum.
  template <class F>
  __device__ __forceinline__ u64 add_up(F f) {
    const int n = (n_chunks + kSuper - 1) / kSuper;
    __syncthreads();
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
    u64 total = 0;
    for (int s = 0; s < n; ++s) total += lds.super[s];
    return total;
  }
  // The least index at which the sum of add_up's weights up to it exceeds r (r below their sum).
  template <class F>
  __device__ __forceinline__ int at_sum(u64 r, F f) {
    constexpr int NW = TH / 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int s = 0;
    while (lds.super[s] <= r) r -= lds.super[s++];
    __syncthreads();
    const int c0 = s * kSuper, c1 = min(c0 + kSuper, n_chunks);
    each(c0, c1, [&](int c, int i, floatx4 v) {
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += f(i + e, v[e]);
      sum = wave_sum(sum);
      if (lane == 0) lds.wave[(c - c0) * NW + w] = sum;
    });
    __syncthreads();
    int at = 0;
    while (lds.wave[at] <= r) r -= lds.wave[at++];
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

  // Of the order of falling logits, rising indexes: the place at which the sum of weights f(logit) reaches
  // `target` (above 0), as its logit and index.  False: all of them come to less.
  template <class F>
  __device__ __forceinline__ bool reach(u64 target, float least, F f, float& at_x, int& at_i) {
    constexpr int PER = kBins / TH;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    float lo = least, hi = m;
    for (;;) {
      // (in 64 bits, where no difference of two logits is lost: hi and lo never share a range)
      const double inv = kBins / ((double)hi - (double)lo);
      auto bin_of = [&](float v) { return min((int)(((double)hi - (double)v) * inv), kBins - 1); };
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i) lds.hist[tid + TH * i] = 0;
      if (tid == 0) lds.bin = -1, lds.count = 0;
      __syncthreads();
      each(0, n_chunks, [&](int, int, floatx4 v) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v[e] >= lo && v[e] <= hi) {
            const u64 x = f(v[e]);
            if (x) atomicAdd(&lds.hist[hi == lo ? 0 : bin_of(v[e])], x);
          }
      });
      __syncthreads();
      u64 own[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += own[i] = lds.hist[PER * tid + i];
      u64 up = wave_scan(sum);
      if (lane == 63) lds.wave[w] = up;
      __syncthreads();
      up -= sum;
      for (int i = 0; i < w; ++i) up += lds.wave[i];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (up < target && target <= up + own[i]) lds.bin = PER * tid + i, lds.before = up;
        up += own[i];
      }
      __syncthreads();
      const int bin = lds.bin;
      if (bin < 0) return false;
      target -= lds.before;
      float most = -INFINITY, fewest = INFINITY;
      each(0, n_chunks, [&](int, int i, floatx4 v) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v[e] >= lo && v[e] <= hi && (hi == lo || bin_of(v[e]) == bin)) {
            most = fmaxf(most, v[e]);
            fewest = fminf(fewest, v[e]);
            const int n = atomicAdd(&lds.count, 1);
            if (n < kList) lds.list_x[n] = v[e], lds.list_i[n] = i + e;
          }
      });
      __syncthreads();
      const int n = lds.count;
      if (n <= kList) {
        for (int i = tid; i < n; i += TH) lds.list_w[i] = f(lds.list_x[i]);
        __syncthreads();
        for (int i = tid; i < n; i += TH) {
          const float v = lds.list_x[i];
          const int index = lds.list_i[i];
          u64 up = 0;
          for (int j = 0; j < n; ++j)
            if (lds.list_x[j] > v || (lds.list_x[j] == v && lds.list_i[j] < index)) up += lds.list_w[j];
          if (up < target && target <= up + lds.list_w[i]) lds.best = i;
        }
        __syncthreads();
        at_x = lds.list_x[lds.best];
        at_i = lds.list_i[lds.best];
        return true;
      }
      hi = block_max(most);
      lo = -block_max(-fewest);
      if (lo == hi) {  // one value: its tokens in the order of their indexes
        const u64 one = f(lo);
        const float v = lo;
        auto same = [v](int, float y) { return (u64)(y == v); };
        add_up(same);
        at_x = v;
        at_i = at_sum((target + one - 1) / one - 1, same);
        return true;
      }
    }
  }
};

template <int TH, int NCH>
__global__ void __launch_bounds__(TH) sample_kernel(SampleArgs a) {
  __shared__ SampleLds lds;
  const int r = blockIdx.x, tid = threadIdx.x;
  Row<TH, NCH> row{a, lds, a.logits + (size_t)r * a.ld, (a.vocab + 4 * TH - 1) / (4 * TH)};
  row.infinite = false;
  if (tid < 64) lds.pow2[tid] = exp2(tid / 64.0);
  const float T = a.temperature ? a.temperature[r] : 1.f, p = a.top_p ? a.top_p[r] : 1.f;
  const float least_p = a.min_p ? a.min_p[r] : 0.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  float most = -INFINITY, least = INFINITY;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) row.held[c] = row.load(c);
  }
  row.each(0, row.n_chunks, [&](int, int, floatx4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      most = fmaxf(most, v[e]);
      if (v[e] > -INFINITY) least = fminf(least, v[e]);
    }
  });
  row.m = row.block_max(most);
  if (row.m == -INFINITY) {  // nothing to choose from
    if (tid == 0) {
      a.tokens[r] = 0;
      if (a.logprob) a.logprob[r] = -INFINITY;
    }
    return;
  }
  least = -row.block_max(-least);
  row.infinite = row.m == INFINITY;
  if (row.infinite) {
    row.m = least = 0.f;
    if constexpr (NCH > 0) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) row.held[c] = row.ordinary(row.held[c]);
    }
  }
  row.frac = a.frac;
  row.scale = 1.4426950408889634 / (double)T;
  const bool greedy = !(T > 0.f) || k == 1 || p <= 0.f;

  // The kept tokens: logits above cut_x, and at cut_x indexes up to cut_i.
  float cut_x = -INFINITY;
  int cut_i = 0x7fffffff;
  auto one = [](float) { return (u64)1; };
  if (greedy) {
    const float m = row.m;
    auto first = [m](int, float v) { return (u64)(v == m); };
    row.add_up(first);
    const int token = row.at_sum(0, first);
    if (tid == 0) {
      a.tokens[r] = token;
      if (a.logprob) a.logprob[r] = 0.f;
    }
    return;
  }
  if (k > 0 && k < a.vocab) row.reach((u64)k, least, one, cut_x, cut_i);
  if (p < 1.f) {
    const float kx = cut_x;
    const int ki = cut_i;
    auto all = [&](int i, float v) { return v > kx || (v == kx && i <= ki) ? row.weight(v) : 0; };
    const u64 mass = row.add_up(all);
    const u64 target = (u64)fmax(ceil((double)p * (double)mass), 1.0);
    row.reach(target, fmaxf(least, kx), [&](float v) { return row.weight(v); }, cut_x, cut_i);
  }
  // w >= min_p, of weights in 64 bits: the nearest unit's is a token's own
  const double floor_y = least_p > 0.f ? log((double)fminf(least_p, 1.f)) : -INFINITY;
  const double inv_t = 1.0 / (double)T;
  const float m = row.m;
  auto kept = [&](int i, float v) {
    const bool in = (v > cut_x || (v == cut_x && i <= cut_i)) && (v == m || ((double)v - (double)m) * inv_t >= floor_y);
    return in ? row.weight(v) : 0;
  };
  const u64 total = row.add_up(kept);
  const double want = (double)(a.u[r] > 0.f ? a.u[r] : 0.f) * (double)total;
  const u64 at = want < (double)total ? (u64)want : total - 1;
  const int token = row.at_sum(at < total ? at : total - 1, kept);
  if (tid == 0) {
    a.tokens[r] = token;
    if (a.logprob) {
      const float v = row.infinite ? 0.f : row.x[token];
      const double y = v == m ? 0.0 : ((double)v - (double)m) * inv_t;
      a.logprob[r] = (float)(y - log(ldexp((double)total, -a.frac)));
    }
  }
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
  auto* kernel = vocab <= 1024 ? sample_kernel<256, 1> : vocab <= 4096 ? sample_kernel<1024, 1> : sample_kernel<1024, 0>;
  const dim3 threads(vocab <= 1024 ? 256 : 1024);
  hipLaunchKernelGGL(kernel, dim3(b), threads, 0, ctx->stream, a);
  AUR_LAUNCH_CHECK(ctx, "sample_kernel");
  return 0;
}
