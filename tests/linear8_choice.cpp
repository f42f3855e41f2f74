// The 8-bit product's planner (laya-cuda_amd/csrc/linear8_plan.hpp) on the problems of standard input: rows, span, slabs, and
// whether gated, 8-bit, of exact products and open to the ring.
#include <cstdio>

#include "linear8_plan.hpp"

int main() {
  laya::Problem8 p;
  int gated, out8, fine, ring;
  while (std::scanf("%lld %lld %d %d %d %d %d", &p.rows, &p.span, &p.slabs, &gated, &out8, &fine, &ring) == 7) {
    p.gated = gated, p.out8 = out8, p.fine = fine, p.ring = ring;
    std::printf("%d\n", laya::linear8_plan(p, 256));
  }
  return 0;
}
