// Every tile of the persistent kernels' walk (laya-cuda_amd/csrc/ring_walk.hpp) is taken exactly once, inside the grid, for
// grids of many shapes, the long and the one-wide among them.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "ring_walk.hpp"

int main() {
  long long checked = 0;
  const int sizes[] = {1, 2, 3, 4, 5, 6, 7, 8, 9, 13, 16, 17, 31, 64, 100, 255, 256, 1000, 4096};
  for (int nx : sizes)
    for (int ny : sizes) {
      const laya::RingWalk w = laya::ring_walk(nx, ny);
      const long long total = static_cast<long long>(nx) * ny;
      if (w.total == 0) {
        if (total * 4 * nx < (1LL << 32)) return std::fprintf(stderr, "refused %d x %d\n", nx, ny), 1;
        continue;
      }
      std::vector<char> seen(total, 0);
      for (int id = 0; id < w.total; ++id) {
        int x = -1, y = -1;
        laya::ring_tile(w, id, &x, &y);
        if (x < 0 || x >= nx || y < 0 || y >= ny || seen[static_cast<long long>(y) * nx + x]++)
          return std::fprintf(stderr, "%d x %d: tile %d at (%d, %d)\n", nx, ny, id, x, y), 1;
        ++checked;
      }
    }
  if (laya::ring_walk(1 << 14, 1 << 14).total || laya::ring_walk(0, 5).total) return 1;
  std::printf("checked %lld\n", checked);
  return 0;
}
