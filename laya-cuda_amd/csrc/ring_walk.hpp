// Which output tile a workgroup of a persistent kernel takes next.  No HIP dependency (tested alone by
// tests/test_ring_walk.py).
#pragma once

#include <cstdint>

namespace laya {

// Workgroups are dealt to the 8 XCDs round-robin, so tile `id`, stepping by a multiple of 8, stays on one.  Each XCD
// takes a contiguous share of the nx x ny tiles, walked in groups of 4 tile rows with the columns outer (`rows`: x
// is the larger operand, and a group's rows of it are fetched into one L2 once), or by whole tile columns.
// `magic` divides by a group's tiles: ceil(2^32 / divisor), exact while total * divisor < 2^32; 0 stands for a
// divisor of one.
struct RingWalk {
  int nx, ny, total, divisor;
  uint32_t magic;
  bool rows;
};

// total is 0 where the walk's division would not be exact.
constexpr RingWalk ring_walk(long long nx, long long ny, bool rows) {
  RingWalk w{};
  const long long divisor = rows ? 4 * nx : ny, total = nx * ny;
  if (nx < 1 || ny < 1 || nx > (1 << 24) || ny > (1 << 24) || total >= (1LL << 31) || total * divisor >= (1LL << 32)) return w;
  w.nx = static_cast<int>(nx);
  w.ny = static_cast<int>(ny);
  w.total = static_cast<int>(total);
  w.divisor = static_cast<int>(divisor);
  w.magic = divisor == 1 ? 0u : static_cast<uint32_t>(((1ULL << 32) + static_cast<unsigned long long>(divisor) - 1) / static_cast<unsigned long long>(divisor));
  w.rows = rows;
  return w;
}

constexpr uint32_t high_product(uint32_t a, uint32_t b) {
  return static_cast<uint32_t>((static_cast<uint64_t>(a) * b) >> 32);
}

// Tile `id` (0 <= id < total).
constexpr void ring_tile(const RingWalk& w, int id, int* x, int* y) {
  const int share = w.total >> 3, rest = w.total & 7, xcd = id & 7;
  const int l = xcd * share + (xcd < rest ? xcd : rest) + (id >> 3);
  const int group = w.magic ? static_cast<int>(high_product(static_cast<uint32_t>(l), w.magic)) : l, in = l - group * w.divisor;
  if (!w.rows) {
    *x = group;
    *y = in;
  } else if (4 * group + 4 <= w.ny) {
    *y = 4 * group + (in & 3);
    *x = in >> 2;
  } else {
    const int size = w.ny - 4 * group;  // 1 .. 3 rows in the last group
    *x = in / size;
    *y = 4 * group + in - *x * size;
  }
}

}  // namespace laya
