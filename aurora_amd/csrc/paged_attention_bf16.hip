// The paged attention's kernels for pools of bf16.
#include "paged_attention.hpp"

namespace aurpaged {

void launch_items_bf16(const MhaArgs& a, const Sizes& z, int p_tile, int tile, unsigned items, hipStream_t st) {
  launch_head<__bf16>(a, p_tile, tile, step_rows(z), items, st);
}

}  // namespace aurpaged
