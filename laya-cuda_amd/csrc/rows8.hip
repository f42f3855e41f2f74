// Kernels that make and read 8-bit rows (rows8.hpp): quantise, read back, and the residual add and norm whose
// output is 8-bit.
//
// All three are bound by HBM: every value is read once and every code written once, and the arithmetic between
// (a maximum over 32 values, one multiplication and one conversion each) hides behind the loads.
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
template <typename T, bool kVec>
__device__ __forceinline__ void store4(T* row, int idx, int width, const float (&v)[4]) {
  if constexpr (kVec) {
    if (idx < width) {
      typename Quad<T>::type t;
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = static_cast<T>(v[i]);
      *reinterpret_cast<typename Quad<T>::type*>(row + idx) = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (idx + i < width) row[idx + i] = static_cast<T>(v[i]);
  }
}

// Writes the codes of quad `idx` (of ld codes a row) and, from a block's first lane, its scale byte.
__device__ __forceinline__ void store_codes(uint8_t* codes, uint8_t* scales, int idx, int ld, const float (&v)[4]) {
  unsigned top = magnitude(v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const unsigned m = magnitude(v[i]);
    top = top > m ? top : m;
  }
  const unsigned s = scale8(block_top8(top));
  if (idx < ld) {
    *reinterpret_cast<unsigned*>(codes + idx) = encode8(v[0], v[1], v[2], v[3], s);
    if ((idx & (kBlock8 - 1)) == 0) scales[idx / kBlock8] = static_cast<uint8_t>(s);
  }
}

// One quad of a row per thread; a wave's 64 quads are 8 whole blocks of one row or of neighbouring rows (rows hold
// whole multiples of 128 codes, 32 quads).
template <typename T, bool kVec>
__global__ __launch_bounds__(256) void quantize8_kernel(Quantize8Args a) {
  const int ld = static_cast<int>(padded8(a.width)), per_row = ld / 4;
  const long long quads = a.rows * per_row, step = static_cast<long long>(gridDim.x) * 256;
  for (long long q = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; q < quads; q += step) {
    const long long row = q / per_row;
    const int idx = static_cast<int>(q - row * per_row) * 4;
    float v[4];
    load4<T, kVec>(static_cast<const T*>(a.x) + row * a.stride, idx, a.width, v);
    store_codes(a.codes + row * ld, a.scales + row * (ld / kBlock8), idx, ld, v);
  }
}

template <typename T, bool kVec>
__global__ __launch_bounds__(256) void dequantize8_kernel(Dequantize8Args a) {
  const int ld = static_cast<int>(padded8(a.width)), per_row = (a.width + 3) / 4;
  const long long quads = a.rows * per_row, step = static_cast<long long>(gridDim.x) * 256;
  for (long long q = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; q < quads; q += step) {
    const long long row = q / per_row;
    const int idx = static_cast<int>(q - row * per_row) * 4;
    const int c = *reinterpret_cast<const int*>(a.codes + row * ld + idx);
    const float s = scale_value8(a.scales[row * (ld / kBlock8) + idx / kBlock8]);
    const float v[4] = {__builtin_amdgcn_cvt_f32_fp8(c, 0) * s, __builtin_amdgcn_cvt_f32_fp8(c, 1) * s,
                        __builtin_amdgcn_cvt_f32_fp8(c, 2) * s, __builtin_amdgcn_cvt_f32_fp8(c, 3) * s};
    store4<T, kVec>(static_cast<T*>(a.out) + row * a.stride, idx, a.width, v);
  }
}

// v = residual + (sum of the branch's partials + bias); y = (v - mean) / sqrt(var + eps) * gamma (+ beta) for
// LayerNorm, y = v / sqrt(mean of v^2 + eps) * gamma for the root-mean-square norm; v goes to sum_out, y to out32 and,
// rounded, to 8-bit rows.  W waves own a row and keep it in registers, C quads a lane: quad c of a lane holds
// elements 256 W c + 256 wave + 4 lane .. +3, so a wave's loads are contiguous and 8 lanes are one block.
// The variance is the centred one, in a second pass over the registers.
template <typename B, int C, int W, bool kVec>
__global__ __launch_bounds__(64 * (W == 1 ? 4 : W)) void norm8_kernel(Norm8Args a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = W == 1 ? blockIdx.x * (blockDim.x >> 6) + wave : blockIdx.x;
  if (row >= a.rows) return;
  const int first = (W == 1 ? 0 : wave * 256) + lane * 4;
  const size_t at = static_cast<size_t>(row) * a.width;
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

  float v[C][4], t[4];
  if (a.branch) {
#pragma unroll
    for (int c = 0; c < C; ++c) load4<B, kVec>(static_cast<const B*>(a.branch) + at, quad(c), a.width, v[c]);
    for (int s = 1; s < a.splits; ++s) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        load4<B, kVec>(static_cast<const B*>(a.branch) + s * a.part_stride + at, quad(c), a.width, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = v[c][i] + t[i];
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
    load4<float, kVec>(a.residual + at, quad(c), a.width, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[c][i] = a.branch ? t[i] + v[c][i] : t[i];
    if (a.sum_out) store4<float, kVec>(a.sum_out + at, quad(c), a.width, v[c]);
  }

  const float n = static_cast<float>(a.width);
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
  const int ld = static_cast<int>(padded8(a.width));
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float g[4], b[4] = {0.f, 0.f, 0.f, 0.f};
    load4<float, kVec>(a.gamma, quad(c), a.width, g);
    if (a.beta) load4<float, kVec>(a.beta, quad(c), a.width, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[c][i] = quad(c) + i < a.width ? v[c][i] * inv * g[i] + b[i] : 0.f;
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

constexpr long long kMaxGrid = 1 << 20;  // of the elementwise kernels; larger problems loop

}  // namespace

hipError_t launch_quantize8(const Quantize8Args& a, DType t, hipStream_t stream) {
  if (a.rows <= 0) return hipSuccess;
  const long long quads = a.rows * (padded8(a.width) / 4);
  const dim3 grid(static_cast<unsigned>(std::min((quads + 255) / 256, kMaxGrid)));
  return for_type(t, [&](auto v) {
    typedef decltype(v) T;
    const bool vec = a.width % 4 == 0 && a.stride % 4 == 0 && aligned(a.x, 4 * sizeof(T));
    if (vec) LAYA_LAUNCH((quantize8_kernel<T, true>), grid, dim3(256), 0, stream, a);
    else LAYA_LAUNCH((quantize8_kernel<T, false>), grid, dim3(256), 0, stream, a);
    return hipGetLastError();
  });
}

hipError_t launch_dequantize8(const Dequantize8Args& a, DType t, hipStream_t stream) {
  if (a.rows <= 0) return hipSuccess;
  const long long quads = a.rows * ((a.width + 3) / 4);
  const dim3 grid(static_cast<unsigned>(std::min((quads + 255) / 256, kMaxGrid)));
  return for_type(t, [&](auto v) {
    typedef decltype(v) T;
    const bool vec = a.width % 4 == 0 && a.stride % 4 == 0 && aligned(a.out, 4 * sizeof(T));
    if (vec) LAYA_LAUNCH((dequantize8_kernel<T, true>), grid, dim3(256), 0, stream, a);
    else LAYA_LAUNCH((dequantize8_kernel<T, false>), grid, dim3(256), 0, stream, a);
    return hipGetLastError();
  });
}

namespace {

template <typename B, bool kVec>
hipError_t launch_norm8_t(const Norm8Args& a, hipStream_t stream) {
  if (a.width <= 2048) {
    const int wpb = a.rows <= 4096 ? 1 : 4;  // few rows: one-wave workgroups, spread over every CU
    const dim3 grid((a.rows + wpb - 1) / wpb), block(64 * wpb);
    switch ((a.width + 255) / 256) {
#define LAYA_CASE(C) case C: LAYA_LAUNCH((norm8_kernel<B, C, 1, kVec>), grid, block, 0, stream, a); break;
      LAYA_CASE(1) LAYA_CASE(2) LAYA_CASE(3) LAYA_CASE(4) LAYA_CASE(5) LAYA_CASE(6) LAYA_CASE(7) LAYA_CASE(8)
#undef LAYA_CASE
    }
  } else {
    const dim3 grid(a.rows), block(256);
    switch ((a.width + 1023) / 1024) {
#define LAYA_CASE(C) case C: LAYA_LAUNCH((norm8_kernel<B, C, 4, kVec>), grid, block, 0, stream, a); break;
      LAYA_CASE(3) LAYA_CASE(4) LAYA_CASE(5) LAYA_CASE(6) LAYA_CASE(7) LAYA_CASE(8)
#undef LAYA_CASE
      default: return hipErrorInvalidValue;
    }
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm8(const Norm8Args& a, DType branch, hipStream_t stream) {
  if (a.rows <= 0) return hipSuccess;
  return for_type(branch, [&](auto v) {
    typedef decltype(v) B;
    const bool vec = a.width % 4 == 0 && aligned(a.residual, 16) && aligned(a.branch, 4 * sizeof(B)) &&
                     (a.splits <= 1 || a.part_stride % 4 == 0) && aligned(a.bias, 16) && aligned(a.gamma, 16) &&
                     aligned(a.beta, 16) && aligned(a.sum_out, 16) && aligned(a.out32, 16);
    return vec ? launch_norm8_t<B, true>(a, stream) : launch_norm8_t<B, false>(a, stream);
  });
}

}  // namespace laya
