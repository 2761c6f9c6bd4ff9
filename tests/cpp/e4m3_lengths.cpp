// How many scales the C++ struct of an 8-bit paged cache makes room for, and which lengths it refuses.
#include "../../aurora_amd/csrc/aurora.hpp"

#include <cstdio>

int main() {
  using Cache = aurora::PagedKvCache<uint8_t>;
  auto refused = [](uint32_t page_len, uint32_t scale_len) {
    try {
      Cache::scales(4, page_len, 2, scale_len);
    } catch (const aurora::Error& e) {
      return e.code;
    }
    return 0;
  };
  const bool ok = Cache::scales(4, 256, 2, 128) == 16 && Cache::scales(4, 16, 2, 1) == 128 && refused(16, 0) == AUR_EINVAL &&
                  refused(16, 32) == AUR_EINVAL && refused(24, 12) == AUR_EINVAL && refused(256, 256) == AUR_ELIMIT;
  std::puts(ok ? "OK" : "wrong");
  return ok ? 0 : 1;
}
