// The 8-bit product's planner (laya-cuda_amd/csrc/linear8_plan.hpp) over problems of all sizes: its tile can make the
// output, and every tile is the choice of some problem.
#include <cstdio>

#include "linear8_plan.hpp"

int main() {
  using namespace laya;
  long long checked = 0, chosen[kRing8 + 1] = {};
  for (long long rows = 1; rows <= 200000; rows += 1 + rows / 6)
    for (long long span = 16; span <= 16384; span += 16 + span / 6)
      for (int slabs = 1; slabs <= 64; slabs += 1 + slabs / 4)
        for (int kind = 0; kind < 16; ++kind) {
          const Problem8 p{rows, span, slabs, (kind & 1) != 0, (kind & 6) == 2, (kind & 6) == 4, (kind & 8) != 0};
          const int id = linear8_plan(p, 256);
          if (id < 0 || id > kRing8 || !tile8_valid(id, p)) return std::fprintf(stderr, "tile %d\n", id), 1;
          ++chosen[id];
          ++checked;
        }
  // 2^30 rows: 2^26 of the smallest tiles, more workgroups than a launch takes, and 2^23 of the largest.
  const Problem8 many{1LL << 30, 16, 1, false, false, true, false}, fewer{(1LL << 30) - 128, 16, 1, false, false, true, false};
  if (tile8_valid(0, many) || linear8_plan(many, 256) != -1 || linear8_plan(fewer, 256) < 11) return std::fprintf(stderr, "2^30 rows\n"), 1;
  for (int id = 0; id <= kRing8; ++id)
    if (!chosen[id]) return std::fprintf(stderr, "tile %d is never chosen\n", id), 1;
  std::printf("checked %lld\n", checked);
  return 0;
}
