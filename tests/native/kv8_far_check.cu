// Host run of the 8-bit cache's tile and slot counts (csrc/kv8.h) at lengths up to the last below 2^31.
#include <cstdio>

#include "../../tiledattention_b200/csrc/kv8.h"

using namespace ta::kv8;

int main() {
  for (int page : {16, 32, 64, 128}) {
    const int64_t most = 0x7fffffffll / page * page;  // capacity of the widest table
    for (int64_t back = 0; back < 1000; ++back) {
      const int length = static_cast<int>(most - back);
      const int64_t want = (static_cast<int64_t>(length) + 127) / 128;
      if (tiles_for(length, 128) != want) {
        std::printf("FAIL tiles_for %d: %d\n", length, tiles_for(length, 128));
        return 1;
      }
      const SeqExtent e = checked_extent(length, 5, 40, most);
      for (int causal : {0, 1})
        if (block_tiles(e, 40, group_reciprocal(1), 0, 128, causal, 128) != want || e.bad) {
          std::printf("FAIL block_tiles %d\n", length);
          return 1;
        }
      const int T = static_cast<int>(0x7fffffffll - back);
      if (slots_for(T, page) != (static_cast<int64_t>(T) + page - 2) / page + 1 || slots_for(T, page) > 0x7fffffffll) {
        std::printf("FAIL slots_for %d\n", T);
        return 1;
      }
    }
  }
  std::printf("ok\n");
  return 0;
}
