// Rotary positions on strided rows of heads, and the frequencies they take.
//
//   angle(row, i) = 2 pi positions[row] turns[i],  (a, b) -> amplitude (a cos - b sin, a sin + b cos)
//
// over the pairs i of each head's leading `rotated` values; what lies behind them is copied.  A value is read and written
// once, so HBM is the bound.  A workgroup takes a few rows: every thread loads its values first, and while they are on their way
// the workgroup makes the rows' cosines and sines once for all heads, in LDS.  The angle is reduced to an eighth of a turn in
// 64 bits (a position of a million at 32 bits would be off by 0.06 radians), the sine and cosine of the rest are fp32.
// 65,536 rows of 32 heads of 64 in bf16: 111 us in a row of such calls, 101 the shortest, 4.8 and 5.3 TB/s (a copy of 4 GiB 4.8; part of it stays in
// the last-level cache), vector instructions 32% of the cycles; 131,072 rows of 10 heads of 128, 131 us and 123.
#include "attend.hpp"

namespace laya {

namespace {

constexpr int kThreads = 256;
// Units a thread has in flight.  Units of 4 bytes and less take more of them for the bytes on their way (heads of 98 in bf16 at
// eight 94 us for 103, of 80 turning 20 values 75 for 90); units of 8 lose by it (heads of 72: 58 us for 54).
constexpr int in_flight(int bytes) { return bytes > 4 ? 4 : 8; }

// n / d from d's rounded inverse: n + 1/2 is exact and the quotient off by at most 2^-23 of itself, less than the 1 / (2 d)
// that lies between it and an integer while n < 2^22.  A workgroup's units are at most a row's 2^20 values.
__device__ __forceinline__ int over(int n, float inverse) { return static_cast<int>((static_cast<float>(n) + 0.5f) * inverse); }

// cos and sin of 2 pi position turns.  The nearest quarter turn goes first, in 64 bits and with one rounding: what is left, at
// most an eighth, rounds to fp32 within 2^-28 of a turn.
__device__ __forceinline__ float2 cos_sin(double position, double turns) {
  const double quarter = rint(position * turns * 4.0);
  const float rest = static_cast<float>(2.0 * fma(position, turns, -0.25 * quarter));  // in half turns, at most 1/4
  const float s = sinpif(rest), c = cospif(rest);
  const int q = static_cast<int>(quarter - 4.0 * floor(quarter * 0.25));
  const float x = q & 1 ? -s : c, y = q & 1 ? c : s;
  return q & 2 ? make_float2(-x, -y) : make_float2(x, y);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// A unit is V pairs (half layout: V values of either half) or V values in a row (interleaved pairs, or values behind the rotated
// ones, which have no pair).  V: the most, up to 16 bytes, that strides, sizes and addresses are multiples of: 67 million values in
// bf16, half layout, at 16 bytes 5.4 TB/s (heads of 64), 8 4.9 (72), 4 4.3 (100), 2 2.8 (98: halves of 49).
// Units below 16 bytes take their indices from inverses, vector instructions being what they wait for; for whole ones that was slower
// (65,536 rows of 32 heads of 64 in bf16 118 us where divisions take 111).
// An interleaved unit may hold both, pairs that turn and values that do not: 114 turned of 128 81 us as units of 4 bytes, 50 as whole ones.
template <typename T, int V, bool kHalf>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 table[];  // [rows][pairs], cosine and sine times the amplitude
  constexpr int kUnits = in_flight(V * sizeof(T));
  constexpr bool kSmall = V * sizeof(T) < 16;
  constexpr int kSide = kHalf ? 1 : (V > 1 ? V : 2);  // values a turning unit takes at one place
  const int pairs = a.rotated / 2;
  const int turning = kHalf ? pairs / V : (a.rotated + kSide - 1) / kSide;  // units of a head that turn
  const int turned = kHalf ? a.rotated : turning * kSide;                   // and the values they hold
  const int copied = a.in_place ? 0 : (a.dim - turned) / V;                 // units that are copied
  const int per_head = turning + copied, per_row = per_head * a.heads;
  const long long row0 = static_cast<long long>(blockIdx.x) * a.rows_each;
  const int rows = static_cast<int>(min(static_cast<long long>(a.rows_each), a.rows - row0));
  const T* x = static_cast<const T*>(a.x);
  T* out = static_cast<T*>(a.out);
  // Units of this workgroup: rows * per_row, shared with the other workgroups of blockIdx.y.
  const int units = rows * per_row;
  bool made = false;
  for (int first = blockIdx.y * kThreads * kUnits; first < units || !made; first += gridDim.y * kThreads * kUnits) {
    Pack<T, V> p[kUnits], q[kUnits];
    long long to[kUnits];
    int pair[kUnits], local[kUnits];  // pair -1: a copied unit, -2: none
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int u = first + k * kThreads + static_cast<int>(threadIdx.x);
      pair[k] = -2;
      if (u < units) {
        const int r = kSmall ? over(u, a.row_inverse) : u / per_row, w = u - r * per_row;
        const int h = kSmall ? over(w, a.head_inverse) : w / per_head, c = w - h * per_head;
        const bool turns = c < turning;
        const int at = turns ? c * (kHalf ? V : kSide) : turned + (c - turning) * V;
        const T* src = x + (row0 + r) * a.x_row + h * a.x_head + at;
        to[k] = (row0 + r) * a.out_row + h * a.out_head + at;
        local[k] = r * pairs;
        pair[k] = turns ? (kHalf ? at : at / 2) : -1;
        p[k] = *reinterpret_cast<const Pack<T, V>*>(src);
        if (turns && (kHalf || V == 1)) q[k] = *reinterpret_cast<const Pack<T, V>*>(src + (kHalf ? pairs : 1));
      }
    }
    if (!made) {
      for (int i = threadIdx.x; i < rows * pairs; i += kThreads) {
        const int r = i / pairs;
        const float2 cs = cos_sin(a.positions[row0 + r], a.turns[i - r * pairs]);
        table[i] = make_float2(cs.x * a.amplitude, cs.y * a.amplitude * a.direction);
      }
      __syncthreads();
      made = true;
    }
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      if (pair[k] == -2) continue;
      if (pair[k] >= 0) {
        const float2* cs = table + local[k] + pair[k];
        if constexpr (kHalf || V == 1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float u = to_float(p[k].v[e]), w = to_float(q[k].v[e]);
            p[k].v[e] = to_half<T>(__builtin_fmaf(u, cs[e].x, -(w * cs[e].y)));
            q[k].v[e] = to_half<T>(__builtin_fmaf(u, cs[e].y, w * cs[e].x));
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            if (V > 2 && 2 * pair[k] + e >= a.rotated) break;  // copied
            const float u = to_float(p[k].v[e]), w = to_float(p[k].v[e + 1]);
            p[k].v[e] = to_half<T>(__builtin_fmaf(u, cs[e / 2].x, -(w * cs[e / 2].y)));
            p[k].v[e + 1] = to_half<T>(__builtin_fmaf(u, cs[e / 2].y, w * cs[e / 2].x));
          }
        }
        if constexpr (kHalf || V == 1) *reinterpret_cast<Pack<T, V>*>(out + to[k] + (kHalf ? pairs : 1)) = q[k];
      }
      *reinterpret_cast<Pack<T, V>*>(out + to[k]) = p[k];
    }
  }
}

// Whether units of V values fit: whole numbers of them, at addresses of their own size.
template <typename T, int V>
bool fits(const RotaryArgs& a) {
  const int size = a.interleaved ? 0 : a.rotated / 2;
  return ((a.x_row | a.x_head | a.out_row | a.out_head | a.dim | size) & (V - 1)) == 0 &&
         ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & (V * sizeof(T) - 1)) == 0;
}

template <typename T, int V, bool kHalf>
hipError_t launch_v(RotaryArgs a, hipStream_t stream) {
  const int pairs = a.rotated / 2;
  const int side = V > 1 ? V : 2, turning = kHalf ? pairs / V : (a.rotated + side - 1) / side;
  const int per_head = turning + (a.in_place ? 0 : (a.dim - (kHalf ? a.rotated : turning * side)) / V);
  const int per_row = per_head * a.heads;
  a.row_inverse = 1.0f / static_cast<float>(per_row);
  a.head_inverse = 1.0f / static_cast<float>(per_head);
  // Rows a workgroup: one batch of units, whose tables fit the 32 KB of LDS that leave a CU five workgroups.  With few rows
  // one each, its units over as many workgroups as hold them (each makes the row's table again).
  const int batch = kThreads * in_flight(V * sizeof(T));
  long long each = batch / per_row;
  if (each > 32768 / (8 * pairs)) each = 32768 / (8 * pairs);
  if (each > a.rows / 1024) each = a.rows / 1024;
  if (each < 1) each = 1;
  a.rows_each = static_cast<int>(each);
  const long long groups = (a.rows + each - 1) / each;
  long long parts = (each * per_row + batch - 1) / batch;
  if (parts > (1LL << 23) / groups) parts = (1LL << 23) / groups;  // a launch of fewer than 2^32 threads; a workgroup takes several batches
  if (parts < 1) parts = 1;
  LAYA_LAUNCH((rotary_kernel<T, V, kHalf>), dim3(static_cast<unsigned>(groups), static_cast<unsigned>(parts)), dim3(kThreads), a.rows_each * pairs * sizeof(float2),
              stream, a);
  return hipGetLastError();
}

template <typename T, int V>
hipError_t launch_t(const RotaryArgs& a, hipStream_t stream) {
  if constexpr (V > 1) {
    if (!fits<T, V>(a)) return launch_t<T, V / 2>(a, stream);
  }
  return a.interleaved ? launch_v<T, V, false>(a, stream) : launch_v<T, V, true>(a, stream);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, DType t, hipStream_t stream) {
  switch (t) {
    case DType::F32: return launch_t<float, 4>(a, stream);
    case DType::F16: return launch_t<f16, 8>(a, stream);
    default: return launch_t<bf16, 8>(a, stream);
  }
}

}  // namespace laya
