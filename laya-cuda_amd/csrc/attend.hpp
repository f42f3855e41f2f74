// Attention over packed sequences with key ranges, capped scores and distance biases: arguments and plan.
#pragma once

#include "attend_plan.hpp"
#include "kernels.hpp"

namespace laya {

constexpr int kMaxSpan = 1024;     // of a bias table: its head's row lies in LDS
constexpr int kMaxAttendDim = 256;

enum class DistanceBias : int { None = 0, Slopes = 1, Table = 2 };

struct AttendArgs : AttendSizes {
  const void *q, *k, *v;
  void* out;
  long long q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;  // elements
  int q_rows, k_rows;
  const int32_t *q_starts, *q_lengths, *k_starts, *k_lengths;  // [n_seq]
  float scale;           // capped: of a raw product, to twice the tanh's argument in log2 units
  float cap;             // in log2 units
  float unit;            // log2 units of a raw product, or, capped, of the tanh's reciprocal: -2 cap
  float per_unit;        // log2(e) / unit: what a bias is multiplied with
  const float* slopes;   // [heads]
  const float* table;    // [heads][2 span + 1]
  int span;
  const int32_t* prefix; // [n_seq] or null
  const int2* bounds;    // [q_rows] (first, end) or null
  // Split plan: row tiles of 32 (token, head) rows, and how many workgroups share a tile's keys.
  int row_tiles, splits;
  float* parts;          // [n_seq][kv_heads][row_tiles][splits][32][dim] sums, then as many [32][2] of reference and total
};

template <int D>  // the compiled head widths
hipError_t launch_attend_dim(const AttendArgs& a, DType t, DistanceBias bias, bool cap, bool split, hipStream_t stream);
hipError_t launch_attend(const AttendArgs& a, DType t, DistanceBias bias, bool cap, const AttendPlan& plan, hipStream_t stream);

struct BoundsArgs {
  const int32_t* documents;  // [rows]
  const int32_t *starts, *lengths;
  int n_seq, rows, max_length;
  int2* bounds;
};
hipError_t launch_document_bounds(const BoundsArgs& a, hipStream_t stream);

struct RotaryArgs {
  const void* x;
  void* out;
  long long x_row, x_head, out_row, out_head;  // elements
  const int32_t* positions;  // [rows]
  const double* turns;       // [rotated / 2] turns a position
  float amplitude, direction;
  long long rows;
  int heads, dim, rotated;
  bool interleaved, in_place;
  int rows_each;             // rows a workgroup, and the inverses of a row's and a head's units (the launcher's)
  float row_inverse, head_inverse;
};
hipError_t launch_rotary(const RotaryArgs& a, DType t, hipStream_t stream);

}  // namespace laya
