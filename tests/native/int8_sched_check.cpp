// The int8 CTA-pair kernel's schedule (csrc/int8_sched.h), checked on the CPU: for
// every problem in range, the planned schedule and the plain ones that a launch
// with fewer resident pairs falls back to compute each (tile, k-block) in exactly
// one work item; a split tile's main pair owns k-blocks [0, kc) and reads exactly
// the slots that its parts write, each written once and by a pair of lower index;
// slots and parts stay within the workspace's. Prints the number of schedules,
// exits 1 on the first violation.
#include <algorithm>
#include <cstdio>
#include <utility>
#include <vector>

#include "../../tt-flow_b200/csrc/int8_sched.h"

using namespace tfb200;

static int fail(const char* what, long m, long n, long k) {
  std::printf("FAIL %s (M=%ld N=%ld K=%ld)\n", what, m, n, k);
  return 1;
}

static int check(const sched::PairSched& s, long m, long n, long k) {
  std::vector<std::vector<std::pair<int, int>>> ranges(s.tiles);
  std::vector<int> writer(s.rem * s.parts, -1), main_of(s.tiles, -1), first(s.tiles, -1);
  std::vector<int> tile_of_slot(s.rem * s.parts, -1);
  for (int p = 0; p < s.pairs; ++p)
    for (int i = 0; i < item_count(s, p); ++i) {
      const PairWork w = item_at(s, p, i);
      if (w.tile < 0 || w.tile >= s.tiles || w.k0 < 0 || w.k0 >= w.k1 || w.k1 > s.kblocks)
        return fail("item range", m, n, k);
      ranges[w.tile].push_back({w.k0, w.k1});
      if (w.role == sched::kPart) {
        if (w.slot < 0 || w.slot >= s.rem * s.parts || writer[w.slot] >= 0) return fail("slot", m, n, k);
        writer[w.slot] = p;
        tile_of_slot[w.slot] = w.tile;
        if (i != item_count(s, p) - 1) return fail("a part that is not its pair's last item", m, n, k);
      } else if (w.role == sched::kMain) {
        if (main_of[w.tile] >= 0 || w.k0 != 0) return fail("main", m, n, k);
        main_of[w.tile] = p;
        first[w.tile] = w.slot;
      } else if (w.k0 != 0 || w.k1 != s.kblocks) {
        return fail("full tile", m, n, k);
      }
    }
  for (int t = 0; t < s.tiles; ++t) {
    std::sort(ranges[t].begin(), ranges[t].end());
    int at = 0;
    for (const auto& r : ranges[t]) {
      if (r.first != at) return fail("coverage", m, n, k);
      at = r.second;
    }
    if (at != s.kblocks) return fail("coverage", m, n, k);
    if ((main_of[t] >= 0) != (ranges[t].size() > 1)) return fail("split without a main pair", m, n, k);
    if (main_of[t] < 0) continue;
    for (int j = 0; j < s.parts; ++j) {
      const int slot = first[t] + j;
      if (slot < 0 || slot >= s.rem * s.parts || tile_of_slot[slot] != t) return fail("main's slots", m, n, k);
      if (writer[slot] >= main_of[t]) return fail("a main pair that waits on a later one", m, n, k);
    }
  }
  return 0;
}

int main() {
  long schedules = 0, split = 0;
  const long ms[] = {1, 128, 129, 257, 300, 513, 900, 1200, 2048, 3000, 4096, 8192, 16000};
  const long ks[] = {1, 128, 129, 384, 1000, 2048, 4096, 5000, 8192, 9001, 16384, 28672, 131071};
  for (const long m : ms)
    for (const long k : ks)
      for (long n = 1; n <= 30000; n += n < 2600 ? 37 : 997) {
        const PairPlan plan = pair_plan(m, n, k);
        const sched::PairSched& s = plan.s;
        if (s.tiles != pair_tiles(m, n, plan.bn) || s.kblocks != (k + kPairBK - 1) / kPairBK)
          return fail("the plan's problem", m, n, k);
        if (s.rem) {
          ++split;
          if (plan.bn != kMaxBN || s.parts < 1 || s.parts > sched::kMaxParts || s.rem * s.parts > s.pairs - s.rem)
            return fail("split", m, n, k);
        }
        if (check(s, m, n, k)) return 1;
        for (const int resident : {kSmPairs, 66, 1}) {
          if (check(sched::plan(s.tiles, s.kblocks, std::min(s.tiles, resident), 0), m, n, k)) return 1;
          ++schedules;
        }
        ++schedules;
      }
  if (!split) return fail("no split schedule in range", 0, 0, 0);
  std::printf("OK %ld schedules, %ld split\n", schedules, split);
  return 0;
}
