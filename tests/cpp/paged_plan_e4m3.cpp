// As paged_plan.cpp, for pools of e4m3.  In: b n_tok max_tok max_own prefix_len n_kv_head group d_head.
#include <cstdio>

#include "../../aurora_amd/csrc/paged_plan.hpp"

int main() {
  aurpaged::Sizes z;
  z.f32 = false;
  z.e4m3 = true;
  while (std::scanf("%d %d %d %d %d %d %d %d", &z.b, &z.n_tok, &z.max_tok, &z.max_own, &z.prefix_len, &z.Hkv, &z.G, &z.dh) ==
         8) {
    const aurpaged::Plan p = aurpaged::make_plan(z);
    std::printf("%d %d %d %d %d %d %d %d %d\n", p.pooled, p.pooled ? p.p_tile : 0, p.p_tiles, p.p_splits, p.o_tile,
                p.o_tiles, p.o_splits, aurpaged::step_rows(z), aurpaged::head_tiles(z.dh));
  }
}
