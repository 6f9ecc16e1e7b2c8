// Output tiles of the int8 CTA-pair kernel (int8_gemm.cu) and their schedule: the
// tile width and the split of a last wave that the launcher takes, and the work
// items that a pair of CTAs runs through. Shared by kernel and launcher, plain C++
// apart from the qualifiers; tests/native/int8_sched_check.cpp checks it on the CPU.
//
// The split differs from the bf16 kernel's (pair_sched.h, whose structure holds it):
// a helper takes one part at most, and int32 parts are exact in any order. What
// holds there holds here: a main pair waits only on pairs with lower indices, which
// the hardware has dispatched before it and which wait on nothing.
#pragma once

#include <cstdint>

#include "pair_sched.h"

namespace tfb200 {

constexpr int kPairBM = 128;   // rows of A per CTA
constexpr int kPairBK = 128;   // k values of a k-block
constexpr int kSmPairs = 74;   // CTA pairs of a B200
constexpr int kMaxBN = 256;    // columns of the widest tile

// Work item i of a pair: the full waves' tiles, then one piece of the split last
// wave. The last `rem` pairs keep k-blocks [0, kc) of its tiles and finish them;
// of the pairs before them, pair g takes part g (tile g / parts).
struct PairWork {
  int tile, k0, k1, role, slot;
};
TFB_SCHED_HD int item_count(const sched::PairSched& s, int p) {
  if (s.rem == 0) return p < s.tiles ? (s.tiles - 1 - p) / s.pairs + 1 : 0;
  return s.waves + (p >= s.pairs - s.rem || p < s.rem * s.parts ? 1 : 0);
}
TFB_SCHED_HD PairWork item_at(const sched::PairSched& s, int p, int i) {
  if (s.rem == 0 || i < s.waves) return {p + i * s.pairs, 0, s.kblocks, sched::kFull, 0};
  const int base = s.waves * s.pairs, r = p - (s.pairs - s.rem);
  if (r >= 0) return {base + r, 0, s.kc, sched::kMain, r * s.parts};
  const int j = p % s.parts, tail = s.kblocks - s.kc;
  return {base + p / s.parts, s.kc + tail * j / s.parts, s.kc + tail * (j + 1) / s.parts, sched::kPart, p};
}

inline int64_t pair_tiles(int64_t m, int64_t n, int bn) {
  return (m + 2 * kPairBM - 1) / (2 * kPairBM) * ((n + bn - 1) / bn);
}

struct PairPlan {
  int bn = kMaxBN;
  sched::PairSched s;
  double cost = 0.0;  // k-blocks
};

// The tile width and schedule over all the pairs of a B200, by an estimate in
// k-blocks of a 256-wide tile (0.3 us). A narrower tile's k-block is hardly
// shorter (A's share of a stage stays, and comes out of L2 for every pair), but
// its epilogue is, so narrow tiles pay where the wide ones leave pairs idle in a
// single short wave; measured, us with 256 / 128 / 64 columns: 256 x 4096 x 4096
// 16.2 / 14.6 / 13.9, 512 x 4096 x 4096 16.5 / 15.5 / 22.5, 200 x 512 x 2048 7.3 /
// 5.7 / 4.8, 1024 x 4096 x 4096 17.7 / 24.8 / 40.0.
// A last wave of R < 74 wide tiles is split when that shortens it: each of its
// tiles keeps k-blocks [0, kc) on one pair, and S parts of the rest go to idle
// pairs, one each. A split costs kSplitCost (writing and handing over the sums,
// clearing the flags) and kReadCost per part, which the finishing pair reads.
// Measured, us without a split / with 1 / 2 / 3 parts: 256 x 16384 x 4096 42.6 /
// 34.5 / 31.8 / 32.3, 1200 x 16384 x 4096 79.8 / 72.0 / 67.8 / 66.8, and where it
// does not pay, 256 x 4096 x 4096 16.1 / 20.2 / 20.9 / 22.6.
constexpr int kSplitCost = 30, kReadCost = 8;
inline PairPlan pair_plan(int64_t m, int64_t n, int64_t k) {
  const int kb = static_cast<int>((k + kPairBK - 1) / kPairBK);
  PairPlan best;
  for (const int bn : {256, 128, 64}) {
    const int64_t tiles = pair_tiles(m, n, bn);
    if (bn < kMaxBN && tiles > 4 * kSmPairs) break;
    const double block = bn == 256 ? 1.0 : bn == 128 ? 0.96 : 0.92, fixed = bn == 256 ? 10.0 : bn == 128 ? 6.0 : 4.0;
    const double cost = static_cast<double>((tiles + kSmPairs - 1) / kSmPairs) * kb * block + fixed;
    if (bn == kMaxBN || cost < best.cost) {
      best.cost = cost;
      best.bn = bn;
      best.s = sched::PairSched();
      best.s.tiles = static_cast<int>(tiles);
      best.s.kblocks = kb;
      best.s.pairs = kSmPairs;
    }
    if (bn < kMaxBN) continue;
    const int rem = best.s.tiles % kSmPairs, idle = kSmPairs - rem;
    for (int parts = 1; rem > 0 && parts <= sched::kMaxParts && rem * parts <= idle; ++parts) {
      // Equal pieces: kc = ceil(KB / (parts + 1)), the parts share the rest.
      const int kc = (kb + parts) / (parts + 1);
      if (kb - kc < parts) break;
      const double split =
          static_cast<double>(best.s.tiles / kSmPairs) * kb + kc + kSplitCost + kReadCost * parts + fixed;
      if (split < best.cost) {
        best.cost = split;
        best.s.waves = best.s.tiles / kSmPairs;
        best.s.rem = rem;
        best.s.parts = parts;
        best.s.kc = kc;
      }
    }
  }
  return best;
}

}  // namespace tfb200
