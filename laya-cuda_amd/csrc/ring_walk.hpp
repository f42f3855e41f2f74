// Which output tile a workgroup of a persistent kernel takes next.  No HIP dependency (tested alone by
// tests/test_ring_walk.py).
#pragma once

#include <cstdint>

namespace laya {

// Workgroups are dealt to the 8 XCDs round-robin, so tile `id`, stepping by a multiple of 8, stays on one.  Each XCD
// takes a contiguous share of the nx x ny tiles, walked in groups of 4 tile rows with the columns outer, so that a
// group's rows of x are fetched into one L2 once and a column's rows of w once a group.  Whole tile columns were faster
// at no shape and 2 to 5% slower at 65,536 x 1,024 x 4,096, 65,536 x 4,096 x 1,024 and 8,192 x 32,768 x 1,024.
// `magic` divides by a group's tiles: ceil(2^32 / divisor), exact while total * divisor < 2^32.
struct RingWalk {
  int nx, ny, total, divisor;
  uint32_t magic;
};

// total is 0 where the walk's division would not be exact.
constexpr RingWalk ring_walk(long long nx, long long ny) {
  RingWalk w{};
  const long long divisor = 4 * nx, total = nx * ny;
  if (nx < 1 || ny < 1 || nx > (1 << 24) || ny > (1 << 24) || total >= (1LL << 31) || total * divisor >= (1LL << 32)) return w;
  w.nx = static_cast<int>(nx);
  w.ny = static_cast<int>(ny);
  w.total = static_cast<int>(total);
  w.divisor = static_cast<int>(divisor);
  w.magic = static_cast<uint32_t>(((1ULL << 32) + static_cast<unsigned long long>(divisor) - 1) / static_cast<unsigned long long>(divisor));
  return w;
}

constexpr uint32_t high_product(uint32_t a, uint32_t b) {
  return static_cast<uint32_t>((static_cast<uint64_t>(a) * b) >> 32);
}

// Tile `id` (0 <= id < total).
constexpr void ring_tile(const RingWalk& w, int id, int* x, int* y) {
  const int share = w.total >> 3, rest = w.total & 7, xcd = id & 7;
  const int l = xcd * share + (xcd < rest ? xcd : rest) + (id >> 3);
  const int group = static_cast<int>(high_product(static_cast<uint32_t>(l), w.magic)), in = l - group * w.divisor;
  if (4 * group + 4 <= w.ny) {
    *y = 4 * group + (in & 3);
    *x = in >> 2;
  } else {
    const int size = w.ny - 4 * group;  // 1 .. 3 rows in the last group; a division would leave the scalar unit
    *x = size == 1 ? in : size == 2 ? in >> 1 : static_cast<int>(high_product(static_cast<uint32_t>(in), 0x55555556u));
    *y = 4 * group + in - *x * size;
  }
}

}  // namespace laya
