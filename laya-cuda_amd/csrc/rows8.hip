// Kernels that make and read 8-bit rows (rows8.hpp): quantise, read back, and the residual add and norm whose
// output is 8-bit.
//
// All three are bound by HBM: every value is read once and every code written once, and the arithmetic between
// (a maximum over 32 values and a conversion each) hides behind the loads.  65,536 rows of 1,024: quantised from fp16
// in 37-39 us (5.3 TB/s) and read back to bf16 in 36, fp32 residual plus bf16 branch normalised in 127 (5.8 TB/s; a copy on this
// card reaches 4.8 past the last-level cache).
#include "rows8.hpp"
#include "kernels.hpp"

#include <algorithm>
#include <type_traits>

namespace laya {

namespace {

template <typename T> struct Quad;
template <> struct Quad<float> { typedef f32x4 type; };
template <> struct Quad<f16> { typedef f16x4 type; };
template <> struct Quad<bf16> { typedef bf16x4 type; };

// Values idx .. idx + 3 of a row, zeros past `width`.  kVec: the row starts and ends on whole quads.
template <typename T, bool kVec>
__device__ __forceinline__ void load4(const T* row, int idx, int width, float (&v)[4]) {
  if constexpr (kVec) {
    if (idx < width) {
      const typename Quad<T>::type t = *reinterpret_cast<const typename Quad<T>::type*>(row + idx);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = idx + i < width ? static_cast<float>(row[idx + i]) : 0.f;
  }
}
// The norm's fp32 outputs, streamed past the caches, which keep the codes for the product that follows (15,088 x 768 with both
// 34.3 -> 27.7 us, 65,536 x 1,024 135 -> 133).
template <typename T, bool kVec>
__device__ __forceinline__ void store4(T* row, int idx, int width, const float (&v)[4]) {
  if constexpr (kVec) {
    if (idx < width) {
      typename Quad<T>::type t;
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = static_cast<T>(v[i]);
      __builtin_nontemporal_store(t, reinterpret_cast<typename Quad<T>::type*>(row + idx));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (idx + i < width) row[idx + i] = static_cast<T>(v[i]);
  }
}

// Writes the codes of quad `idx` (of ld codes a row) and, from a block's first lane, its scale byte.
__device__ __forceinline__ void store_codes(uint8_t* codes, uint8_t* scales, int idx, int ld, const float (&v)[4]) {
  const unsigned s = scale8(block_top8(magnitude(largest(largest(0.f, v[0], v[1]), v[2], v[3]))));
  if (idx < ld) {
    *reinterpret_cast<unsigned*>(codes + idx) = encode8(v[0], v[1], v[2], v[3], s);
    if ((idx & (kBlock8 - 1)) == 0) scales[idx / kBlock8] = static_cast<uint8_t>(s);
  }
}

// Quantising and reading back work on pieces of 16 bytes of values: kPiece<T> of them a thread, 4 or 8, so that a block
// is 8 or 4 lanes.  A workgroup owns 256 U pieces, all loaded before the first is used.  Piece q of the matrix is
// piece q % per_row of row q / per_row; the workgroup's first one is divided in 64 bits, once, the others by a
// multiplication.  What many pieces leave is streamed past the caches: 65,536 x 1,024 16-bit values quantised in 38.4 instead
// of 42.6 us, and with the product that reads the codes behind it in the same time; values read back always are, that many in
// 30.6 instead of 39.9 us.  Fewer codes are kept for their product: quantising and 512 x 1,024 x 4,096 17.3 -> 16.5 us, 15,088 x
// 2,304 x 768 74.8 -> 73.4.
template <typename T> constexpr int kPiece = 16 / sizeof(T);
struct Place8 {
  long long row;
  int piece;
};
__device__ __forceinline__ Place8 place8(long long row0, int in, int per_row, unsigned magic) {
  // in < per_row + 1024: at most one row further for long rows, else divided exactly (in and per_row are under 2^11).
  const int rows = per_row >= 1024 ? (in >= per_row) : static_cast<int>(__umulhi(static_cast<unsigned>(in), magic));
  return Place8{row0 + rows, in - rows * per_row};
}
// Pieces a thread: one of up to 2^21 pieces (their workgroups run in few rounds: 5,003 x 1,000 fp32 values take 6.3 us,
// and 6.9 with four), four of more (65,536 x 1,024 fp16 values: 57 us with one, 42 with four).
int pieces_a_thread(long long pieces) { return pieces <= 1 << 21 ? 1 : 4; }
unsigned piece_magic(int per_row) {  // ceil(2^32 / per_row); rows hold 16 pieces at least
  return static_cast<unsigned>(((1ULL << 32) + per_row - 1) / per_row);
}

template <typename T, bool kVec, int U>
__global__ __launch_bounds__(256) void quantize8_kernel(Quantize8Args a, unsigned magic) {
  constexpr int E = kPiece<T>;
  typedef T TE __attribute__((ext_vector_type(E)));
  const int ld = static_cast<int>(padded8(a.width)), per_row = ld / E;
  const long long total = a.rows * per_row, first = static_cast<long long>(blockIdx.x) * (256 * U);
  const long long row0 = first / per_row;
  const int in0 = static_cast<int>(first - row0 * per_row) + threadIdx.x;
  float v[U][E];
  Place8 o[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    o[u] = place8(row0, in0 + u * 256, per_row, magic);
    if (first + u * 256 + threadIdx.x >= total) continue;
    const T* const src = static_cast<const T*>(a.x) + o[u].row * a.stride + o[u].piece * E;
    const int left = a.width - o[u].piece * E;
    if constexpr (kVec) {
      TE t;
      if (left > 0) t = *reinterpret_cast<const TE*>(src);
#pragma unroll
      for (int i = 0; i < E; ++i) v[u][i] = left > 0 ? static_cast<float>(t[i]) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[u][i] = i < left ? static_cast<float>(src[i]) : 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (first + u * 256 + threadIdx.x >= total) return;  // rows are whole blocks: alike in a block's lanes
    float widest = 0.f;
#pragma unroll
    for (int i = 0; i < E; i += 2) widest = largest(widest, v[u][i], v[u][i + 1]);
    unsigned top = magnitude(widest);
#pragma unroll
    for (int d = 1; d < kBlock8 / E; d <<= 1) {
      const unsigned m = __shfl_xor(top, d, kWave);
      top = top > m ? top : m;
    }
    const unsigned s = scale8(top);
    typedef unsigned Codes __attribute__((ext_vector_type(E / 4)));
    Codes c;
#pragma unroll
    for (int i = 0; i < E / 4; ++i) c[i] = encode8(v[u][4 * i], v[u][4 * i + 1], v[u][4 * i + 2], v[u][4 * i + 3], s);
    Codes* const dst = reinterpret_cast<Codes*>(a.codes + o[u].row * ld + o[u].piece * E);
    if constexpr (U > 1) __builtin_nontemporal_store(c, dst);
    else *dst = c;
    if ((threadIdx.x & (kBlock8 / E - 1)) == 0)
      a.scales[o[u].row * (ld / kBlock8) + o[u].piece / (kBlock8 / E)] = static_cast<uint8_t>(s);
  }
}

template <typename T, bool kVec, int U>
__global__ __launch_bounds__(256) void dequantize8_kernel(Dequantize8Args a, unsigned magic) {
  constexpr int E = kPiece<T>;
  typedef int Codes __attribute__((ext_vector_type(E / 4)));
  typedef T TE __attribute__((ext_vector_type(E)));
  const int ld = static_cast<int>(padded8(a.width)), per_row = ld / E;
  const long long total = a.rows * per_row, first = static_cast<long long>(blockIdx.x) * (256 * U);
  const long long row0 = first / per_row;
  const int in0 = static_cast<int>(first - row0 * per_row) + threadIdx.x;
  Codes c[U];
  unsigned s[U];
  Place8 o[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    o[u] = place8(row0, in0 + u * 256, per_row, magic);
    if (first + u * 256 + threadIdx.x >= total) continue;
    c[u] = *reinterpret_cast<const Codes*>(a.codes + o[u].row * ld + o[u].piece * E);
    s[u] = a.scales[o[u].row * (ld / kBlock8) + o[u].piece / (kBlock8 / E)];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (first + u * 256 + threadIdx.x >= total) return;
    const float f = scale_value8(s[u]);
    float v[E];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      v[4 * i] = __builtin_amdgcn_cvt_f32_fp8(c[u][i], 0) * f;
      v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(c[u][i], 1) * f;
      v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(c[u][i], 2) * f;
      v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(c[u][i], 3) * f;
    }
    T* const dst = static_cast<T*>(a.out) + o[u].row * a.stride + o[u].piece * E;
    const int left = a.width - o[u].piece * E;
    if constexpr (kVec) {
      TE t;
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] = static_cast<T>(v[i]);
      if (left > 0) __builtin_nontemporal_store(t, reinterpret_cast<TE*>(dst));
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i < left) dst[i] = static_cast<T>(v[i]);
    }
  }
}

// v = residual + (sum of the branch's partials + bias); y = (v - mean) / sqrt(var + eps) * gamma (+ beta) for
// LayerNorm, y = v / sqrt(mean of v^2 + eps) * gamma for the root-mean-square norm; v goes to sum_out, y to out32 and,
// rounded, to 8-bit rows.  W waves own a row and keep it in registers, C quads a lane: quad c of a lane holds
// elements 256 W c + 256 wave + 4 lane .. +3, so a wave's loads are contiguous and 8 lanes are one block.
// The variance is the centred one, in a second pass over the registers.  A workgroup is one row: four rows a workgroup
// took up to 7% longer.
// NS: the branch's partials when they are known at launch, so that they, the residual and the parameters are loaded
// before the first addition (one memory round trip); -1: any number, in a loop, and the rest where it is used.  An fp32
// residual of 512 x 1,024 with a bf16 branch: 4.1 us early, 5.0 late; 65,536 x 1,024: 127 and 132.
template <typename B, int C, int W, bool kVec, int NS>
__global__ __launch_bounds__(64 * W) void norm8_kernel(Norm8Args a) {
  constexpr bool kEarly = NS > 0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x;
  const int first = wave * 256 + lane * 4;
  auto quad = [&](int c) { return first + c * 256 * W; };
  __shared__ float part[W];
  auto row_sum = [&](float v) {
    v = wave_sum(v);
    if constexpr (W > 1) {
      __syncthreads();  // the previous sum has been read
      if (lane == 0) part[wave] = v;
      __syncthreads();
      v = part[0];
#pragma unroll
      for (int w = 1; w < W; ++w) v = v + part[w];
    }
    return v;
  };
  const float n = static_cast<float>(a.width);
  const int ld = static_cast<int>(padded8(a.width));
  float gamma[kEarly ? C : 1][4], beta[kEarly ? C : 1][4];
  if constexpr (kEarly) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      load4<float, kVec>(a.gamma, quad(c), a.width, gamma[c]);
      if (a.beta) load4<float, kVec>(a.beta, quad(c), a.width, beta[c]);
    }
  }
  const size_t at = static_cast<size_t>(row) * a.width;
  float v[C][4], t[4], res[kEarly ? C : 1][4];
  if constexpr (kEarly) {
#pragma unroll
    for (int c = 0; c < C; ++c) load4<float, kVec>(a.residual + at, quad(c), a.width, res[c]);
  }
  if (a.branch) {
#pragma unroll
    for (int c = 0; c < C; ++c) load4<B, kVec>(static_cast<const B*>(a.branch) + at, quad(c), a.width, v[c]);
    if constexpr (NS > 1) {
      float p[NS - 1][C][4];
#pragma unroll
      for (int s = 1; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < C; ++c)
          load4<B, kVec>(static_cast<const B*>(a.branch) + s * a.part_stride + at, quad(c), a.width, p[s - 1][c]);
#pragma unroll
      for (int s = 1; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[c][i] = v[c][i] + p[s - 1][c][i];
    } else if constexpr (NS < 0) {
      for (int s = 1; s < a.splits; ++s) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          load4<B, kVec>(static_cast<const B*>(a.branch) + s * a.part_stride + at, quad(c), a.width, t);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[c][i] = v[c][i] + t[i];
        }
      }
    }
    if (a.bias) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        load4<float, kVec>(a.bias, quad(c), a.width, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = v[c][i] + t[i];
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int r = kEarly ? c : 0;
    if constexpr (!kEarly) load4<float, kVec>(a.residual + at, quad(c), a.width, res[0]);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[c][i] = a.branch ? res[r][i] + v[c][i] : res[r][i];
    if (a.sum_out) store4<float, kVec>(a.sum_out + at, quad(c), a.width, v[c]);
  }

  if (!a.rms) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) s += v[c][i];
    const float mean = row_sum(s) / n;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[c][i] = quad(c) + i < a.width ? v[c][i] - mean : 0.f;
  }
  float sq = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) sq += v[c][i] * v[c][i];
  const float inv = 1.0f / sqrtf(row_sum(sq) / n + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = kEarly ? c : 0;
    if constexpr (!kEarly) {
      load4<float, kVec>(a.gamma, quad(c), a.width, gamma[0]);
      if (a.beta) load4<float, kVec>(a.beta, quad(c), a.width, beta[0]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = v[c][i] * inv * gamma[p][i];
      v[c][i] = quad(c) + i >= a.width ? 0.f : a.beta ? y + beta[p][i] : y;
    }
    if (a.out32) store4<float, kVec>(a.out32 + at, quad(c), a.width, v[c]);
    store_codes(a.codes + static_cast<size_t>(row) * ld, a.scales + static_cast<size_t>(row) * (ld / kBlock8), quad(c), ld, v[c]);
  }
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename F>
hipError_t for_type(DType t, F&& f) {
  switch (t) {
    case DType::F16: return f(f16());
    case DType::BF16: return f(bf16());
    default: return f(0.f);
  }
}

}  // namespace

hipError_t launch_quantize8(const Quantize8Args& a, DType t, hipStream_t stream) {
  if (a.rows <= 0) return hipSuccess;
  return for_type(t, [&](auto v) {
    typedef decltype(v) T;
    const int per_row = static_cast<int>(padded8(a.width) / kPiece<T>), u = pieces_a_thread(a.rows * per_row);
    const long long groups = (a.rows * per_row + 256 * u - 1) / (256 * u);
    const dim3 grid(static_cast<unsigned>(groups));
    const unsigned magic = piece_magic(per_row);
    const bool vec = a.width % kPiece<T> == 0 && a.stride % kPiece<T> == 0 && aligned(a.x, 16);
    if (vec && u == 4) LAYA_LAUNCH((quantize8_kernel<T, true, 4>), grid, dim3(256), 0, stream, a, magic);
    else if (vec) LAYA_LAUNCH((quantize8_kernel<T, true, 1>), grid, dim3(256), 0, stream, a, magic);
    else if (u == 4) LAYA_LAUNCH((quantize8_kernel<T, false, 4>), grid, dim3(256), 0, stream, a, magic);
    else LAYA_LAUNCH((quantize8_kernel<T, false, 1>), grid, dim3(256), 0, stream, a, magic);
    return hipGetLastError();
  });
}

hipError_t launch_dequantize8(const Dequantize8Args& a, DType t, hipStream_t stream) {
  if (a.rows <= 0) return hipSuccess;
  return for_type(t, [&](auto v) {
    typedef decltype(v) T;
    const int per_row = static_cast<int>(padded8(a.width) / kPiece<T>), u = pieces_a_thread(a.rows * per_row);
    const long long groups = (a.rows * per_row + 256 * u - 1) / (256 * u);
    const dim3 grid(static_cast<unsigned>(groups));
    const unsigned magic = piece_magic(per_row);
    const bool vec = a.width % kPiece<T> == 0 && a.stride % kPiece<T> == 0 && aligned(a.out, 16);
    if (vec && u == 4) LAYA_LAUNCH((dequantize8_kernel<T, true, 4>), grid, dim3(256), 0, stream, a, magic);
    else if (vec) LAYA_LAUNCH((dequantize8_kernel<T, true, 1>), grid, dim3(256), 0, stream, a, magic);
    else if (u == 4) LAYA_LAUNCH((dequantize8_kernel<T, false, 4>), grid, dim3(256), 0, stream, a, magic);
    else LAYA_LAUNCH((dequantize8_kernel<T, false, 1>), grid, dim3(256), 0, stream, a, magic);
    return hipGetLastError();
  });
}

namespace {

template <typename B, bool kVec, int NS>
hipError_t launch_norm8_t(const Norm8Args& a, hipStream_t stream) {
  const dim3 grid(a.rows);
#define LAYA_CASE(C, W) \
  if (a.width <= 256 * W * C) { LAYA_LAUNCH((norm8_kernel<B, C, W, kVec, NS>), grid, dim3(64 * W), 0, stream, a); return hipGetLastError(); }
  LAYA_CASE(1, 1) LAYA_CASE(2, 1) LAYA_CASE(3, 1) LAYA_CASE(4, 1) LAYA_CASE(5, 1) LAYA_CASE(6, 1) LAYA_CASE(8, 1)
  LAYA_CASE(3, 4) LAYA_CASE(4, 4) LAYA_CASE(6, 4) LAYA_CASE(8, 4)
#undef LAYA_CASE
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_norm8(const Norm8Args& a, DType branch, hipStream_t stream) {
  if (a.rows <= 0) return hipSuccess;
  return for_type(branch, [&](auto v) {
    typedef decltype(v) B;
    const bool vec = a.width % 4 == 0 && aligned(a.residual, 16) && aligned(a.branch, 4 * sizeof(B)) &&
                     (a.splits <= 1 || a.part_stride % 4 == 0) && aligned(a.bias, 16) && aligned(a.gamma, 16) &&
                     aligned(a.beta, 16) && aligned(a.sum_out, 16) && aligned(a.out32, 16);
    const int splits = a.branch ? a.splits : 1;
    if (!vec) return launch_norm8_t<B, false, -1>(a, stream);
    // Eight quads a lane of everything are registers that many rows' waves miss, unless fp32 partials keep HBM busy
    // anyhow: 8,192 x 8,192 with a bf16 branch 177 us early, 154 late (fp32: 199 and 209), 512 rows 11.4 and 12.9.
    const bool early = a.width <= 6144 || sizeof(B) == 4 || a.rows <= 512;
    if (early && splits == 1) return launch_norm8_t<B, true, 1>(a, stream);
    if constexpr (sizeof(B) == 4) {  // split-K partials are fp32: 16,384 x 2,048 with four 152 us, in the loop 160
      if (early && splits == 2) return launch_norm8_t<B, true, 2>(a, stream);
      if (early && splits == 3) return launch_norm8_t<B, true, 3>(a, stream);
      if (early && splits == 4) return launch_norm8_t<B, true, 4>(a, stream);
    }
    return launch_norm8_t<B, true, -1>(a, stream);
  });
}

}  // namespace laya
