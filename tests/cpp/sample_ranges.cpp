// Reads lines "m T bin" and "m T p -1" and prints, for the border of range `bin` or of min_p = p, the logit, whether
// it passes, whether the next smaller float does, and how many logits were looked at.
#include "../../aurora_amd/csrc/sample_ranges.hpp"

#include <cmath>
#include <cstdio>

using namespace aursample;

int main() {
  float m, T, p;
  int bin;
  while (std::scanf("%f %f %f %d", &m, &T, &p, &bin) == 4) {
    const Ranges r = first_ranges(m, T);
    const double floor_y = std::log((double)p), inv_t = 1.0 / (double)T;
    int looked = 0;
    auto passes = [&](float v) {
      ++looked;
      return bin >= 0 ? r.of(v) <= bin : v >= m || ((double)v - (double)m) * inv_t >= floor_y;
    };
    const double c = bin >= 0 ? r.hi - (bin + 0.5) / r.inv : (double)m + (double)T * floor_y;
    const float at = bin >= 0 ? r.edge(bin) : least_kept(m, T, floor_y);
    const float same = least_passing(c > kLeastLogit ? std::fmin((float)c, m) : kLeastLogit, m, passes);
    const int n = looked;
    const bool ends = at <= kLeastLogit || !passes(std::nextafterf(at, -INFINITY));
    std::printf("%a %d %d %d\n", at, same == at && passes(at), ends, n);
  }
}
