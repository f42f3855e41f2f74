// Which tile an 8-bit product takes.  No HIP dependency (tested alone by tests/test_linear8_plan.py).
#pragma once

namespace laya {

// BM x BN outputs a workgroup, WM x WN waves times KG groups that split the slabs, S stages of SL slabs; FAST: the 8-bit
// matrix unit, else widened codes.  Then the fit that linear8_plan uses, in microseconds, from products of 64 to 1,024
// tiles and K = 512 to 4,096 with operands that alternate between three sets (out of L2): a launch takes
// L + rounds (B + C slabs), a round being OCC tiles a CU.  Tiles of two a CU hide one workgroup's fill and epilogue
// behind the other's slabs, which pays from the second round on.
//            ID   BM   BN WM WN KG SL  S  FAST  OCC  L     B     C
#define LAYA_LINEAR8_TILES                                             \
  LAYA_T(0, 16, 16, 1, 1, 8, 8, 4, false, 1, 1.4f, 2.45f, 0.086f)      \
  LAYA_T(1, 16, 32, 1, 1, 8, 8, 3, false, 1, 1.4f, 3.09f, 0.108f)      \
  LAYA_T(2, 16, 64, 1, 2, 4, 4, 3, false, 1, 1.6f, 2.56f, 0.202f)      \
  LAYA_T(3, 64, 32, 2, 1, 4, 4, 3, false, 1, 1.6f, 2.90f, 0.275f)      \
  LAYA_T(4, 64, 64, 2, 2, 2, 2, 4, false, 1, 1.6f, 2.91f, 0.471f)      \
  LAYA_T(5, 64, 64, 2, 2, 2, 2, 4, true, 1, 1.4f, 3.02f, 0.334f)       \
  LAYA_T(6, 64, 64, 2, 2, 1, 1, 4, false, 2, 1.7f, 3.10f, 0.810f)      \
  LAYA_T(7, 64, 64, 2, 2, 1, 1, 4, true, 2, 1.7f, 2.40f, 0.690f)       \
  LAYA_T(8, 64, 128, 2, 4, 1, 1, 4, true, 1, 1.7f, 3.02f, 0.565f)      \
  LAYA_T(9, 128, 128, 2, 4, 1, 1, 4, true, 1, 2.3f, 4.53f, 0.791f)     \
  LAYA_T(10, 128, 128, 2, 4, 1, 1, 2, true, 2, 4.4f, 3.70f, 1.400f)    \
  LAYA_T(11, 128, 128, 2, 4, 1, 1, 4, false, 1, 2.8f, 4.44f, 1.229f)   \
  LAYA_T(12, 128, 128, 2, 2, 1, 1, 2, false, 2, 4.0f, 6.20f, 2.280f)
// The persistent rings come last: on the 8-bit matrix unit, and with exact products.
constexpr int kLinear8Tiles = 13, kFastRing8 = kLinear8Tiles, kRing8 = kLinear8Tiles + 1;

struct Tile8Cost {
  int bm, bn;
  bool fast;
  int occ;
  float l, b, c;
};
constexpr Tile8Cost kTile8Costs[] = {
#define LAYA_T(ID, BM, BN, WM, WN, KG, SL, S, FAST, OCC, L, B, C) {BM, BN, FAST, OCC, L, B, C},
    LAYA_LINEAR8_TILES
#undef LAYA_T
};
static_assert(sizeof(kTile8Costs) / sizeof(kTile8Costs[0]) == kLinear8Tiles, "a row per tile");

struct Problem8 {
  long long rows, span;  // output rows, and columns with an 8-bit row's padding
  int slabs;             // of 128 codes
  bool gated, out8, fine, ring;  // 8-bit outputs; `fine`: exact products alone; `ring`: the ring kernels take this call
};

// Workgroups of BM x BN tiles.
constexpr long long tiles8(const Problem8& p, long long bm, long long bn) {
  const long long oc = p.gated ? bn / 2 : bn;
  return (p.span + oc - 1) / oc * ((p.rows + bm - 1) / bm);
}

// Whether tile `id` can make this output: a block of 32 output codes and a group of 16 gate and 16 value rows lie
// inside one tile, exact products are made where they are asked for, and a launch has fewer than 2^32 threads.
constexpr bool tile8_valid(int id, const Problem8& p) {
  if (id == kFastRing8 || id == kRing8) return p.ring && p.slabs >= 2 && !(p.fine && id == kFastRing8);
  if (id < 0 || id >= kLinear8Tiles) return false;
  const Tile8Cost& t = kTile8Costs[id];
  return !(p.fine && t.fast) && !(p.gated && t.bn % 32) && !(p.out8 && (p.gated ? t.bn / 2 : t.bn) % 32) &&
         tiles8(p, t.bm, t.bn) < (1LL << 32) / 512;
}

// The valid tile with the least estimated time on `cus` compute units.
constexpr int linear8_plan(const Problem8& p, int cus) {
  int best = -1;
  float least = 0.f;
  for (int id = 0; id <= kRing8; ++id) {
    if (!tile8_valid(id, p)) continue;
    const bool ring = id >= kLinear8Tiles;
    const long long tiles = ring ? tiles8(p, 256, 256) : tiles8(p, kTile8Costs[id].bm, kTile8Costs[id].bn);
    const float n = static_cast<float>(p.slabs);
    float time = 0.f;
    if (ring) {
      // Its first round depends on how many CUs fetch and store at once.
      const float full = tiles < cus ? static_cast<float>(tiles) / static_cast<float>(cus) : 1.f;
      const long long rounds = (tiles + cus - 1) / cus;
      time = id == kRing8 ? 12.4f + full + n * (2.56f + 0.5f * full) + static_cast<float>(rounds - 1) * (15.3f + 3.27f * n)
                          : 6.6f + 5.5f * full + n * (1.34f + 0.36f * full) + static_cast<float>(rounds - 1) * (5.4f + 1.7f * n);
    } else {
      const Tile8Cost& t = kTile8Costs[id];
      const long long round = static_cast<long long>(cus) * t.occ, rounds = (tiles + round - 1) / round;
      // Up to one tile a CU, a second place on it goes unused.
      const float share = tiles <= cus && t.occ == 2 ? 0.75f : 1.f;
      time = t.l + static_cast<float>(rounds) * share * (t.b + t.c * n);
    }
    if (best < 0 || time < least) {
      best = id;
      least = time;
    }
  }
  return best;
}

}  // namespace laya
