// Host-side planning of the 8-bit layer's kernels (csrc/plan.h), run over whole ranges of sizes on the CPU.
#include <cstdio>
#include <cstring>

#include "plan.h"

using namespace b2g;

// Every ring that ring_shape() allows fits the shared memory that its kernel may ask for, and its blocks
// together fit an SM (228 KB, of which each block costs 1 KB beside its own).
static int ring() {
  constexpr long long kStatic = 544;  // the kernels' words: float buf[128], a flag, rounding
  long long tried = 0;
  for (int most = 1; most <= 28; ++most)
    for (uint32_t stage = 16; stage <= 300000; stage += 16) {
      int blocks = 0, stages = 0;
      if (!ring_shape(stage, most, &blocks, &stages)) continue;
      ++tried;
      const long long bytes = ring_bytes(stages, stage);
      if (bytes != stages * (stage + 8ll)) return printf("stage %u: %d stages take %lld bytes\n", stage, stages, bytes), 1;
      if (bytes > kRingSmem || stages < 2 || stages > 4 || blocks < 1 || blocks > most ||
          blocks * (bytes + kStatic + 1024) > 228 * 1024)
        return printf("stage %u, at most %d blocks: %d blocks of %d stages, %lld bytes each\n", stage, most, blocks, stages, bytes), 1;
    }
  printf("ok %lld\n", tried);
  return 0;
}

int main(int argc, char** argv) {
  if (argc > 1 && !strcmp(argv[1], "ring")) return ring();
  return 2;
}
