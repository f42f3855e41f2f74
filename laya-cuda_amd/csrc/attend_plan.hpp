// Which kernel an attention call over packed sequences takes, and in how many workgroups.  No HIP dependency (tested alone by
// tests/test_attend_plan.py).
#pragma once

#include <algorithm>
#include <cmath>

namespace laya {

constexpr int kPlannedUnits = 256;  // compute units that plans are made for: workspaces are told without a device, and any plan is right on any card
constexpr int kMaxSplits = 64;  // of a sequence's keys over workgroups: one lane each when they are joined

struct AttendSizes {
  int heads, kv_heads, group, dim;  // group = heads / kv_heads
  int n_seq, max_q, max_k;
  int before, after;                // -1: no limit
  bool prefixed;
};

// The launch of a call: which kernel, and for the split one its row tiles and splits; workspace in bytes.
struct AttendPlan {
  bool split;
  int row_tiles, splits;
  long long workspace;
};
enum AttendKernel : int { kAttendPlanned = 0, kAttendMany = 1, kAttendFew = 2 };

// Which kernel: by what either takes, in us, as fitted to both on 18 calls of one to 64 sequences, 48 to 1,000 queries and 64 to
// 8,000 keys.  A prompt's workgroup takes its blocks one after the other (1.0 us each for heads of 64 with one on a CU, 1.5 with
// two; 1.4 for heads of 128); a tile of few rows shares them among eight waves, at 2 us (4) for each tile that a CU has and 0.1 us
// (0.2) a block of 32.  The prompts' kernel, the other: 512 tokens of 12 heads of 64 14.9 and 8.4 us, 4 such 13.0 and 16.5, 1,024 of 16
// heads 20.2 and 15.0, 2 x 2,048 52.6 and 71.2; 512 of 32 heads of 128 behind 8,000 keys 171 and 96, 1,000 causal ones 29 and 41.
// Heads above 128 run prompts in workgroups of 256 queries and few rows in four waves, and go by the same formulas: over 75 calls of heads of
// 160, 192 and 256 the choice takes 1.01 times the better kernel's time on average, at most 1.16 (chosen and other: 4 x 512 tokens of 8 heads of 256 37.1
// and 32.0 us, 2,048 causal ones of 16 heads of 160 on 4 88 and 77; 4,096 causal ones of 8 heads of 160 135 and 142, of 256 168 and 188).
// Lengths are not known here: splits go by max_k and the number of tiles, however uneven the sequences are.
inline AttendPlan attend_plan(const AttendSizes& a, int kernel) {
  AttendPlan p{};
  const long long few = static_cast<long long>(a.max_q) * a.group;
  p.row_tiles = static_cast<int>((few + 31) / 32);
  p.splits = 1;
  // Keys that a tile's queries see: at most, and on average where later queries see more.
  double most = a.max_k;
  if (a.before >= 0 && !a.prefixed) most = std::min(most, a.before + (a.after >= 0 ? a.after : a.max_k) + 96.0);
  const double mean = a.after >= 0 && a.max_k == most ? most - 0.5 * std::min(a.max_q, a.max_k) : most;
  const double base = static_cast<double>(a.n_seq) * a.kv_heads * p.row_tiles;
  // As many workgroups as compute units, each with a block of keys for every wave at least; joining costs what two such
  // rounds take, so two workgroups a tile are not worth it.
  const double n = std::floor(std::min(kPlannedUnits / std::max(base, 1.0), most / 256.0));
  if (n >= 3) p.splits = static_cast<int>(std::min<double>(n, kMaxSplits));
  const double prompt = static_cast<double>((a.max_q + 127) / 128) * a.n_seq * a.heads / kPlannedUnits;  // workgroups a CU
  const double wide = a.dim <= 64 ? 1 : a.dim <= 128 ? 2 : a.dim / 64.0;
  const double prompt_us = 5.5 + (prompt > 1 ? mean : most) / 64 * (wide == 1 ? std::max(1.0, 0.55 + 0.5 * prompt) : wide / 2 * std::max(1.4, 0.3 + prompt));
  const double split_us = 5 + (p.splits > 1 ? 3 : 0) + std::max(1.0, base * p.splits / kPlannedUnits) * wide * (2 + 0.1 * mean / p.splits / 32);
  p.split = kernel == kAttendPlanned ? split_us < prompt_us : kernel == kAttendFew;
  if (!p.split) p.splits = 1;
  if (p.splits > 1) p.workspace = static_cast<long long>(base) * p.splits * 32 * (a.dim + 2) * 4;
  return p;
}

// Workgroups of the kernel for few rows.  units: the (sequence, key head) pairs, where the tiles of each stay on one XCD, and pairs count
// as whole rounds of 8; else 0.
struct FewGrid {
  long long groups;
  int units;
};
inline FewGrid few_grid(const AttendSizes& a, int row_tiles, int splits) {
  const long long units = static_cast<long long>(a.n_seq) * a.kv_heads, share = (units + 7) / 8;
  // Evenly over the XCDs, or in one round on each however unevenly.
  const bool kept = row_tiles > 1 && splits == 1 && (share * 56 <= units * 8 || share * row_tiles <= (a.dim <= 64 ? 64 : 32));
  return {(kept ? share * 8 : units) * row_tiles * splits, kept ? static_cast<int>(units) : 0};
}

}  // namespace laya
