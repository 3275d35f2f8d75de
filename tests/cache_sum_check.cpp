// Host replay of the sum that sizes the chunks of the attention over a paged
// cache (htree_cache_index.h), up to as many requests as a call takes: times the
// units wanted, a chunk is never below the exact number of tiles, which the
// workspace is sized for.  The lengths are those that a sum in fp32 loses most
// of: one long request per lane before many short ones.
// Test infrastructure: built and run by tests/test_cache_sum.py on the CPU.
#include <cstdio>
#include <random>
#include <vector>

#include "htree_cache_index.h"

using namespace htree;

int main() {
  std::mt19937 g(3);
  int fails = 0, calls = 0;
  for (int B : {1, 64, 65, 1000, kCacheMaxRequests})
    for (int kind = 0; kind < 4; ++kind) {
      const int KT = 16, cap = 1 << 30, target = kind % 2 ? 512 : 256, G = 1, R = 16;
      // tokens of a request, one new one each
      const auto len = [&](int b) -> int {
        if (kind == 0) return 16 * (1 + b % 5);
        if (kind == 1) return b < 64 ? cap : 16;  // 2^26 tiles first: one more is an eighth of a step of fp32
        if (kind == 2) return b < 64 ? cap : 16 * 5;
        return (int)((uint32_t)b * 2654435761u % (uint32_t)cap);
      };
      float lanes[64];
      __int128 exact = 0;
      for (int b = 0; b < B; ++b) exact += draft_tiles(draft_req(b, b + 1, len(b), B), cap, KT);
      for (int l = 0; l < 64; ++l)
        lanes[l] = draft_lane_tiles(l, B, cap, KT, G, R, [&](int b) { return draft_req(b, b + 1, len(b), B); });
      // the lanes' tree, in fp32
      for (int m = 1; m < 64; m <<= 1)
        for (int l = 0; l < 64; l += 2 * m) lanes[l] += lanes[l + m];
      const int chunk = draft_chunk(lanes[0], target);
      // (a chunk of more tiles than a request can have: nothing is split)
      const bool good = chunk > cap / KT || (__int128)chunk * target >= exact;
      ++calls;
      if (!good) {
        ++fails;
        std::printf("FAIL B %d kind %d: chunk %d x %d below %lld\n", B, kind, chunk, target, (long long)exact);
      }
      // and not far above it: the units fill the GPU
      if (chunk < 1 << 30 && (double)chunk * target > (double)exact * 1.001 + 5.0 * target) {
        ++fails;
        std::printf("FAIL B %d kind %d: chunk %d x %d far above %lld\n", B, kind, chunk, target, (long long)exact);
      }
    }
  std::printf("%d calls, %d failures\n", calls, fails);
  return fails != 0;
}
