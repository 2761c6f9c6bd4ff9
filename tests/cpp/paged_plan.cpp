// Prints how the paged attention cuts calls into items (aurora_amd/csrc/paged_plan.hpp), one line a call.
// In: b n_tok max_tok max_own prefix_len n_kv_head group d_head f32.  Out: pooled p_tile p_tiles p_splits
// o_tile o_tiles o_splits, rows of a step's own items, 16-column tiles of a head.
#include <cstdio>

#include "../../aurora_amd/csrc/paged_plan.hpp"

int main() {
  aurpaged::Sizes z;
  int f32;
  while (std::scanf("%d %d %d %d %d %d %d %d %d", &z.b, &z.n_tok, &z.max_tok, &z.max_own, &z.prefix_len, &z.Hkv, &z.G,
                    &z.dh, &f32) == 9) {
    z.f32 = f32 != 0;
    const aurpaged::Plan p = aurpaged::make_plan(z);
    std::printf("%d %d %d %d %d %d %d %d %d\n", p.pooled, p.pooled ? p.p_tile : 0, p.p_tiles, p.p_splits, p.o_tile,
                p.o_tiles, p.o_splits, aurpaged::step_rows(z), aurpaged::head_tiles(z.dh));
  }
}
