// Host harness for sine_share.h: for tokens of every number of threads, that those of each workgroup form
// each of its tokens' pairs once; prints "OK", or the first that is not.
#include <cstdio>
#include <vector>

#include "backend/mi355x/sine_share.h"

using namespace txk;

int main() {
  for (uint32_t tt = 1; tt <= 1100; ++tt) {
    const uint32_t per = tt <= 256 ? 256 / tt : 1, blocks = tt <= 256 ? 1 : (tt + 255) / 256;
    for (uint32_t half : {1u, 5u, 16u, 38u, 64u, 128u, 300u, 2048u})
      for (uint32_t block = 0; block < blocks; ++block) {
        std::vector<int> times(per * half, 0);
        for (uint32_t t = 0; t < 256; ++t) {
          // thread t's token of the workgroup, and its place among that token's
          const uint32_t token = tt <= 256 ? t / tt : 0, in = tt <= 256 ? t % tt : 256 * block + t;
          if (token >= per || in >= tt)
            continue;
          const SineShare s = sine_share(t, tt, in);
          if (s.token != token || s.step < 1) {
            printf("threads %u: thread %u of workgroup %u has token %u, step %u\n", tt, t, block, s.token, s.step);
            return 1;
          }
          for (uint32_t i = s.first; i < half; i += s.step)
            ++times[s.token * half + i];
        }
        for (size_t i = 0; i < times.size(); ++i)
          if (times[i] != 1) {
            printf("threads %u, pairs %u: workgroup %u forms pair %zu %d times\n", tt, half, block, i, times[i]);
            return 1;
          }
      }
  }
  puts("OK");
}
