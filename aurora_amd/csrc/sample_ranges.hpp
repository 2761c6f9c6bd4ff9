// The ranges of logits that a choice of tokens is made by, and the logits at which they and min_p's kept tokens end:
// arithmetic alone, for the device and for a look at it without one.
#pragma once

#include <cstdint>

namespace aursample {

constexpr int kBins = 1024;
constexpr float kLeastLogit = -3.402823466e38f;  // that can be chosen

// To the nearest whole number by adding 1.5·2^52, whose sum has it in its last bits.
constexpr double kWhole = 6755399441055744.0;
constexpr __attribute__((always_inline)) inline int low32(double x) {
  return (int)(uint32_t)__builtin_bit_cast(uint64_t, x);
}

// Floats (zeros of both signs, no NaN) as whole numbers of the same order, without gaps; the way back is the same.
constexpr int order_of(int bits) { return bits ^ ((bits >> 31) & 0x7fffffff); }
constexpr int order_of(float x) { return order_of(__builtin_bit_cast(int, x)); }
constexpr float at_order(int i) { return __builtin_bit_cast(float, order_of(i)); }

// The least logit that passes, where with one all larger ones up to `most` do, which does.  The guess is hardly ever
// more than a float away, but where the border is 0, up to 2^30 floats stand between two results of a difference
// of two logits: so by steps that double until the border lies between two of them, and then by halves.
template <class P>
constexpr float least_passing(float guess, float most, P passes) {
  const int first = order_of(kLeastLogit), last = order_of(most);
  int low = order_of(guess), up = low;  // passes not, and passes
  if (passes(guess)) {
    for (unsigned step = 1;; step *= 2) {
      low = (unsigned)up - (unsigned)first < step ? first - 1 : (int)((unsigned)up - step);
      if (low < first || !passes(at_order(low))) break;
      up = low;
    }
  } else {
    for (unsigned step = 1;; step *= 2) {
      up = (unsigned)last - (unsigned)low <= step ? last : (int)((unsigned)low + step);
      if (up == last || passes(at_order(up))) break;
      low = up;
    }
  }
  while ((unsigned)up - (unsigned)low > 1) {
    const int mid = (int)((unsigned)low + ((unsigned)up - (unsigned)low) / 2);
    (passes(at_order(mid)) ? up : low) = mid;
  }
  return at_order(up);
}

// Ranges below hi, 1 / inv wide; all below the last one share it.
struct Ranges {
  double hi, inv;
  constexpr __attribute__((always_inline)) int of(float v) const {
    return low32(__builtin_fmin((hi - (double)v) * inv, kBins - 1.0) + kWhole);
  }
  // The least logit of the ranges 0 .. bin.
  constexpr __attribute__((always_inline)) float edge(int bin) const {
    if (bin >= kBins - 1) return kLeastLogit;
    const double c = hi - (bin + 0.5) / inv;
    const float most = (float)hi, guess = c > kLeastLogit ? ((float)c < most ? (float)c : most) : kLeastLogit;
    return least_passing(guess, most, [this, bin](float v) { return of(v) <= bin; });
  }
};
// The first ranges of a histogram below the largest logit m: kBins of them down to where weights end.
constexpr Ranges first_ranges(float m, float T) { return {m, kBins / (32.0 * (double)T)}; }

// The least logit that min_p keeps of a row with the largest one m: kept are m and (x − m) / T >= floor_y.
constexpr __attribute__((always_inline)) inline float least_kept(float m, float T, double floor_y) {
  const double inv_t = 1.0 / (double)T, c = (double)m + (double)T * floor_y;
  const float guess = c > kLeastLogit ? ((float)c < m ? (float)c : m) : kLeastLogit;
  return least_passing(guess, m, [=](float v) { return v >= m || ((double)v - (double)m) * inv_t >= floor_y; });
}

}  // namespace aursample
