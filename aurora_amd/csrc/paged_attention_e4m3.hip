// The paged attention's kernels for pools of e4m3 with a scale for each block of tokens and head.
#include "paged_attention.hpp"

namespace aurpaged {

void launch_items_e4m3(const MhaArgs& a, const Sizes& z, int p_tile, int tile, unsigned items, hipStream_t st) {
  launch_head<e4m3>(a, p_tile, tile, step_rows(z), items, st);
}

}  // namespace aurpaged
