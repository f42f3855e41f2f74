// Which tile an 8-bit product takes.  No HIP dependency (tested alone by tests/test_linear8_plan.py).
#pragma once

namespace laya {

// BM x BN outputs a workgroup, WM x WN waves times KG groups that split the slabs, S stages of SL slabs; FAST: the 8-bit
// matrix unit, else widened codes.  Then the fit that linear8_plan uses, in microseconds (tune_linear8_costs.py sweeps, fits and
// checks it): a launch takes L + rounds (B + C slabs), a round being OCC tiles a CU.  On 120 held-out products the choice
// takes at most 1.04 times the best tile of exact products, at most 1.16 times the best of all, and on average under 1.005.
// Tiles of two a CU hide one workgroup's fill and epilogue behind the other's slabs, which pays from the second round on.
//            ID   BM   BN WM WN KG SL  S  FAST  OCC  L     B     C
#define LAYA_LINEAR8_TILES                                             \
  LAYA_T(0, 16, 16, 1, 1, 8, 8, 4, false, 1, 1.13f, 2.77f, 0.083f)     \
  LAYA_T(1, 16, 32, 1, 1, 8, 8, 3, false, 1, 1.20f, 3.34f, 0.119f)     \
  LAYA_T(2, 16, 64, 1, 2, 4, 4, 3, false, 1, 1.21f, 3.17f, 0.198f)     \
  LAYA_T(3, 64, 32, 2, 1, 4, 4, 3, false, 1, 0.68f, 4.06f, 0.256f)     \
  LAYA_T(4, 64, 64, 2, 2, 2, 2, 4, false, 1, 0.32f, 3.85f, 0.439f)     \
  LAYA_T(5, 64, 64, 2, 2, 2, 2, 4, true, 1, 0.24f, 3.90f, 0.270f)      \
  LAYA_T(6, 64, 64, 2, 2, 1, 1, 4, false, 2, 1.56f, 3.15f, 0.798f)     \
  LAYA_T(7, 64, 64, 2, 2, 1, 1, 4, true, 2, 1.53f, 3.04f, 0.553f)      \
  LAYA_T(8, 64, 128, 2, 4, 1, 1, 4, true, 1, 0.17f, 4.01f, 0.492f)     \
  LAYA_T(9, 128, 128, 2, 4, 1, 1, 4, true, 1, 0.00f, 5.79f, 0.717f)    \
  LAYA_T(10, 128, 128, 2, 4, 1, 1, 2, true, 2, 0.00f, 6.95f, 1.097f)   \
  LAYA_T(11, 128, 128, 2, 4, 1, 1, 4, false, 1, 0.00f, 5.52f, 1.233f)  \
  LAYA_T(12, 128, 128, 2, 2, 1, 1, 2, false, 2, 1.48f, 8.39f, 1.900f)
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

// The rings': start, what every CU's fetching and storing at once adds to it, a slab of the first round, a further round, its
// slabs.
constexpr float kFastRingCost[] = {6.72f, 3.51f, 1.48f, 6.74f, 1.55f};
constexpr float kRingCost[] = {8.84f, 1.97f, 2.71f, 9.65f, 2.62f};

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
      const float full = tiles < cus ? static_cast<float>(tiles) / static_cast<float>(cus) : 1.f;
      const long long rounds = (tiles + cus - 1) / cus;
      const float* const k = id == kRing8 ? kRingCost : kFastRingCost;
      time = k[0] + k[1] * full + k[2] * n + static_cast<float>(rounds - 1) * (k[3] + k[4] * n);
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
