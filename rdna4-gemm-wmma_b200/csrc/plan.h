// Launch planning: tile shape and K splitting of the tensor-core GEMM, and the shape of the row
// kernels' rings.  Pure host functions of the problem's sizes and the GPU's SM count, shared by the
// launchers (b2g_api.cu, b2g_q8.cu, b2g_rows.cu), b2g_plan_preview and the CPU tests that pin them.
#pragma once
#include <algorithm>
#include <cstdint>

namespace b2g {

struct TileChoice {
  int cg;    // CTAs per tile (1 or 2)
  int bn;    // tile width in columns (128, 256 or 512)
  bool half; // CG = 2 half-height pair tile: 128 x 256 over the pair, 64 A rows per CTA
};

// Fraction of the resident CTA groups that `units` work units keep busy over their waves.
inline double wave_fill(int64_t units, int64_t groups) {
  groups = std::max<int64_t>(1, groups);
  const int64_t waves = (units + groups - 1) / groups;
  return (double)units / (double)(std::max<int64_t>(1, waves) * groups);
}

// Split count when every tile of a small problem is split (fewer than half as many tiles as
// CTA groups): at most 8 one-CTA splits or 4 half-height pair splits (the largest cluster of
// the cluster fix-up is 8 CTAs), 16 for pairs, each split keeping at least 16 K blocks.  One-CTA
// tiles may keep 8 K blocks a split instead, when that fills strictly more CTA groups
// (measured on B200: 1024^3 in two splits of 8 blocks, 512x512x2048 and 256x1024x2048 in four,
// 5-22% faster than with 16).  *short_split tells whether the 8-block rule was taken.
inline int64_t small_splits(int64_t tiles, int64_t kit, int64_t groups, int cg, bool half,
                            bool* short_split = nullptr) {
  if (short_split) *short_split = false;
  if (2 * tiles > groups) return 1;
  const int64_t cap = half ? 4 : (cg == 1 ? 8 : 16);
  const int64_t per = std::max<int64_t>(1, groups / std::max<int64_t>(1, tiles));
  const int64_t sp16 = kit >= 32 ? std::max<int64_t>(1, std::min<int64_t>({per, kit / 16, cap})) : 1;
  if (cg != 1 || half || kit < 16) return sp16;
  const int64_t sp8 = std::max<int64_t>(1, std::min<int64_t>({per, kit / 8, cap}));
  if (wave_fill(tiles * sp8, groups) > wave_fill(tiles * sp16, groups) + 1e-9) {
    if (short_split) *short_split = true;
    return sp8;
  }
  return sp16;
}

// nmt: 128-row M tiles; kit: K blocks of one tile; sms: SMs; opt_cg / opt_bn: forced values
// (0 = choose); opt_rows: 64 = half-height pair tiles whenever the shape allows, 0 or 128 =
// never (the planner does not choose them: measured on B200 they stream B more slowly than
// one-CTA tiles on every skinny shape tried, although their split-K reduction is smaller).
inline TileChoice choose_tiles(int64_t nmt, int64_t N, int64_t kit, int sms, int opt_cg,
                               int opt_bn, int opt_rows = 0) {
  int cg = opt_cg, bn = opt_bn;
  if (bn == 128) cg = 1;  // the 128-column tile exists for one CTA only
  const bool half_ok = (bn == 0 || bn == 256) && cg != 1;
  if (opt_rows == 64 && half_ok) return {2, 256, true};
  const int64_t pairs = std::max(1, sms / 2);
  if (cg != 1 && cg != 2) {
    // Small problems (fewer 128x256 tiles than SMs).  When split-K applies, one-CTA tiles (the
    // cluster fix-up), of the width whose work units (tiles times the split count) fill the
    // SMs best; on a tie the 128x256 tile, which moves a quarter fewer bytes per FLOP.  When
    // no width splits, 256x256 pair tiles if they fill the SMs as well: the same CTAs, each
    // loading half as many B bytes per FLOP (measured on B200: 2048^3 and 4096x1024x4096
    // 10-15% faster than 128x256 one-CTA tiles).
    if (bn == 0 && nmt * ((N + 255) / 256) < sms) {
      auto fill = [&](int w, int64_t* splits, bool* short_split) {
        const int64_t tiles = nmt * ((N + w - 1) / w);
        const int64_t sp = small_splits(tiles, kit, sms, 1, false, short_split);
        *splits = sp;
        return wave_fill(tiles * sp, sms);
      };
      int64_t sp128 = 1, sp256 = 1;
      bool s128 = false, s256 = false;
      const double f128 = fill(128, &sp128, &s128), f256 = fill(256, &sp256, &s256);
      if (sp128 == 1 && sp256 == 1 && nmt >= 2 &&
          wave_fill(((nmt + 1) / 2) * ((N + 255) / 256), pairs) >= std::max(f128, f256) - 1e-9)
        return {2, 256, false};
      cg = 1;
      // on a tie, the width that needs no 8-block splits (measured: 4096x512x1024 unsplit
      // 128x128 tiles beat 128x256 tiles in two splits of 8 blocks), then 128x256
      if (f128 > f256 + 1e-9 || (f128 > f256 - 1e-9 && s256 && !s128))
        bn = 128;
      else
        bn = 256;
    } else {
      cg = (nmt >= 2) ? 2 : 1;
    }
  }
  if (bn != 128 && bn != 256 && bn != 512) {
    // 512-wide pair tiles pull a quarter fewer operand bytes from L2 per FLOP; use them when
    // there are enough of them to fill every CTA pair at least twice, or when their waves fill
    // the pairs as well as 256-wide tiles' do (measured on B200: 2048x4096x4096, 3072^3 and
    // 4096x4096x2048 10-13% faster with one or two waves of 512-wide tiles).
    const int64_t mp = (nmt + 1) / 2;
    const int64_t t512 = mp * ((N + 511) / 512), t256 = mp * ((N + 255) / 256);
    bn = (cg == 2 && (t512 >= 2 * pairs || wave_fill(t512, pairs) >= wave_fill(t256, pairs) - 1e-9))
             ? 512
             : 256;
  }
  if (cg == 1 && bn == 512) bn = 256;  // one CTA: at most 256 columns (two accumulators)
  if (cg == 2 && bn == 128) bn = 256;
  return {cg, bn, false};
}

struct SplitChoice {
  int num_full;     // tiles done as one unit over all of K (the first ones in tile order)
  int k_splits;     // units per remaining tile
  int k_per_split;  // K blocks per split unit
};

// Split-K for under-filled grids and for the tail wave.  group_cap: CTA groups resident at
// once (SMs, or CTA pairs); opt_split: forced split count (0 = choose); half: half-height pair
// tiles (at most 4 splits, and never a tail split: they split only with the cluster fix-up).
inline SplitChoice choose_splits(int num_tiles, int k_iters, int group_cap, int cg, int opt_split,
                                 bool tail_split, bool half = false) {
  int splits = opt_split;
  int full = 0;
  if (splits <= 0) {
    splits = 1;
    full = num_tiles;
    const int waves = num_tiles / std::max(1, group_cap);
    const int rem = num_tiles - waves * group_cap;
    // Every tile split when the tiles fill at most half the CTA groups (small_splits: each
    // split keeps 16 K blocks, or 8 for one-CTA tiles when that fills more groups; below that
    // the fixed cost of a unit, pipeline fill, partial write and fix-up, outweighs the shorter
    // main loop).
    const int64_t sp = small_splits(num_tiles, k_iters, group_cap, cg, half);
    if (sp > 1) {
      splits = (int)sp;
      full = 0;
    } else if (!half && tail_split && waves >= 1 && rem > 0 && group_cap / rem >= 2 &&
               k_iters >= 32) {
      // whole waves plus a partial one: split only the partial wave's tiles
      splits = std::min({group_cap / rem, 4, k_iters / 16});
      full = waves * group_cap;
    }
  }
  splits = std::max(1, std::min(splits, std::max(1, k_iters)));
  SplitChoice c;
  c.k_per_split = (k_iters + splits - 1) / splits;
  c.k_splits = c.k_per_split > 0 ? (k_iters + c.k_per_split - 1) / c.k_per_split : 1;  // no empty split
  if (c.k_splits < 1) c.k_splits = 1;
  c.num_full = c.k_splits == 1 ? num_tiles : full;
  return c;
}

// A product whose accumulators may sum at most `part` K blocks each (fp32 weight gradients: the tensor
// core's accumulator truncates).  Whole tiles take their K in parts within one launch; where K is split
// over CTAs, every launch has at most `part` blocks a split, and the next one adds to it.  Tiles
// and splits are chosen once, for all of K: every launch takes them as they are.
struct PartPlan {
  TileChoice tile;
  int splits;      // of every tile in every launch
  int64_t blocks;  // K blocks of a launch (the last one may have fewer)
};

// Tiles as choose_tiles, but at most 256 columns where K goes in parts (two accumulators in TMEM).
inline TileChoice choose_part_tiles(int64_t nmt, int64_t cols, int64_t kit, int sms, int opt_cg, int opt_bn,
                                    int64_t part) {
  const TileChoice tc = choose_tiles(nmt, cols, kit, sms, opt_cg, opt_bn, 128);
  if (part > 0 && kit > part && tc.bn == 512) return {tc.cg, 256, false};
  return tc;
}

// group_cap: CTA groups of `tile` resident at once; opt_split: forced split count (0 = choose).
inline PartPlan plan_parts(const TileChoice& tile, int64_t nmt, int64_t cols, int64_t kit, int group_cap,
                           int opt_split, int64_t part) {
  const int64_t tiles = (nmt + tile.cg - 1) / tile.cg * ((cols + tile.bn - 1) / tile.bn);
  const int splits = choose_splits((int)tiles, (int)kit, group_cap, tile.cg, opt_split, false).k_splits;
  if (splits == 1) return {tile, 1, kit};
  // Launches of equal length.  Where two splits would need several launches, whole tiles in parts are
  // faster (us, graph: 2048 tokens, dW 1024 x 2048 29.5 against 34.0, 4096 x 2048 x 1024 46.3 against
  // 51.4); with four splits they are not (4096 x 1024 x 1024 44.8 against 38.0).
  const int64_t most = splits * part, launches = std::max<int64_t>(1, (kit + most - 1) / most);
  if (splits == 2 && launches > 1 && opt_split <= 0) return {tile, 1, kit};
  return {tile, splits, (kit + launches - 1) / launches};
}

// K blocks of one part of a whole tile's kit blocks.
inline int part_length(int kit, int part) {
  const int parts = (kit + part - 1) / part;
  return (kit + parts - 1) / parts;
}

// Dynamic shared memory that the row kernels' rings may ask for: what a block can have, less the kernels'
// static words.
constexpr uint32_t kRingSmem = 222 * 1024;
// Bytes of a ring of `stages` buffers of `stage` bytes, each with its barrier.
inline uint32_t ring_bytes(int stages, uint32_t stage) { return (uint32_t)stages * (stage + 8); }

// Stages and blocks an SM of a ring kernel: as many blocks as `most` if two stages of each fit (one
// block's copies run while another's row is worked on), then up to four stages.  False where not
// even two stages of one block fit.
inline bool ring_shape(uint32_t stage, int most, int* blocks, int* stages) {
  constexpr uint32_t kPerBlock = 2048;  // of each block: static words, what the driver keeps, rounding
  for (int n = most; n >= 1; --n) {
    const uint32_t fit = ((kRingSmem + kPerBlock) / n - kPerBlock) / (stage + 8);
    if (fit >= 2) {
      *blocks = n;
      *stages = (int)std::min<uint32_t>(4, fit);
      return true;
    }
  }
  return false;
}

}  // namespace b2g
