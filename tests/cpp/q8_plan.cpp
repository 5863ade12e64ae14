// Host-side planning of the 8-bit layer's kernels (csrc/plan.h), run over whole ranges of sizes on the CPU.
#include <cstdio>
#include <cstring>

#include "plan.h"
#include "sched.h"

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

// No accumulator of an fp32 weight gradient sums more than 12 K blocks (768 tokens), whatever the sizes
// and the forced tile or split, and the launches cover every block once.
static int parts() {
  constexpr int kPart = 12;
  static const int opts[][3] = {{0, 0, 0}, {1, 0, 0}, {2, 0, 0}, {1, 128, 0}, {2, 512, 0}, {0, 0, 1}, {0, 0, 3}, {2, 256, 16}, {1, 0, 64}};
  long long tried = 0, split = 0;
  for (const auto& o : opts)
    for (int sms : {148, 132, 74})
      for (long long rows = 64; rows <= 8192; rows += 128)
        for (long long cols = 64; cols <= 8192; cols += 128)
          for (long long tokens : {1, 64, 700, 769, 1000, 1536, 1537, 2048, 3000, 4096, 5000, 8192, 16384, 20001, 65536}) {
            const int64_t nmt = (rows + 127) / 128, kit = (tokens + 63) / 64;
            const TileChoice tile = choose_part_tiles(nmt, cols, kit, sms, o[0], o[1], kPart);
            const PartPlan p = plan_parts(tile, nmt, cols, kit, sms / tile.cg, o[2], kPart);
            const int tiles = (int)((nmt + tile.cg - 1) / tile.cg * ((cols + tile.bn - 1) / tile.bn));
            int64_t worst = 0, done = 0;
            ++tried;
            for (int64_t b = 0; b < kit; b += p.blocks) {  // as the launches are made
              const int k = (int)std::min(p.blocks, kit - b);
              const SplitChoice s = choose_splits(tiles, k, sms / tile.cg, tile.cg, p.splits, false);
              const int sum = s.k_splits > 1 ? s.k_per_split : k > kPart ? part_length(k, kPart) : k;
              if (s.k_splits > 1 && s.num_full != 0) return printf("a whole tile beside split ones\n"), 1;
              if (s.k_splits == 1 && k > kPart && p.tile.bn == 512) return printf("parts in a 512-column tile\n"), 1;
              worst = std::max<int64_t>(worst, sum);
              done += k;
              split += s.k_splits > 1;
            }
            if (worst > kPart || done != kit)
              return printf("%lld tokens, dW %lld x %lld, options %d %d %d: %lld blocks in one accumulator, %lld of %lld done\n", tokens,
                            rows, cols, o[0], o[1], o[2], (long long)worst, (long long)done, (long long)kit), 1;
          }
  printf("ok %lld, %lld split launches\n", tried, split);
  return 0;
}

// The words that the aligning copy reads without a check lie inside the matrix, for every row, base
// alignment, length and pitch.
static int words() {
  long long tried = 0;
  for (int base = 4; base < 8; ++base)
    for (int rows = 1; rows <= 12; ++rows)
      for (int bytes = 1; bytes <= 40; ++bytes)
        for (int pitch = bytes; pitch <= bytes + 9; ++pitch)
          for (int r = 0; r < rows; ++r) {
            if (!b2g_row_words_inside(r, rows, pitch)) continue;
            const int row = base + r * pitch, first = row & ~3, last = (row + bytes - 1) | 3;  // first and last byte read
            const int end = base + (rows - 1) * pitch + bytes;
            ++tried;
            if (first < base || last >= end)
              return printf("base %d, row %d of %d, %d bytes, pitch %d: reads [%d, %d] of [%d, %d)\n", base, r, rows, bytes, pitch, first,
                            last, base, end), 1;
          }
  // and the rows in the middle of an ordinary matrix go without the check
  for (int r = 1; r < 99; ++r)
    if (!b2g_row_words_inside(r, 100, 3)) return printf("row %d of 100 is checked\n", r), 1;
  printf("ok %lld\n", tried);
  return 0;
}

int main(int argc, char** argv) {
  if (argc > 1 && !strcmp(argv[1], "ring")) return ring();
  if (argc > 1 && !strcmp(argv[1], "parts")) return parts();
  if (argc > 1 && !strcmp(argv[1], "words")) return words();
  return 2;
}
