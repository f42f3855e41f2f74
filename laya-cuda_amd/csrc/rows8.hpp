// 8-bit rows: e4m3 codes with one power-of-two scale per 32 of them.
//
// A row of `width` values is stored as padded8(width) codes, a multiple of 128 (the codes past the width are
// zeros), and one scale byte s per 32 codes; code c of the block stands for e4m3(c) * 2^(s - 127).  The scale is
// the smallest one that leaves the whole block within the largest code, 448 (at most 247); a block of zeros has s = 0, and
// a block that holds a NaN or an infinity has s = 255 and reads back as NaNs.  128 codes are what one
// v_mfma_scale_f32_16x16x128_f8f6f4 takes of a row, and their four scale bytes are one aligned dword.
//
// Power-of-two scales cost up to one bit of the codes' range against a scale of amax / 448, but no rounding:
// reading back is exact, and a producer whose amax moves by one unit in the last place changes no value by more
// than a code's rounding.
#pragma once

#include "common.hpp"

namespace laya {

constexpr int kBlock8 = 32;      // codes that share a scale
constexpr int kPad8 = 128;       // codes per row are a multiple of this
constexpr unsigned kInf = 0x7f800000u;
__host__ __device__ constexpr long long padded8(long long width) { return (width + kPad8 - 1) / kPad8 * kPad8; }

// Magnitude bits: as unsigned integers they order like the magnitudes, with NaNs above infinity.
__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }
// The largest of top (>= 0 or NaN), |a| and |b|: one v_maximum3_f32, which keeps NaNs (fmaxf drops them).
__device__ __forceinline__ float largest(float top, float a, float b) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, __builtin_fabsf(a)), __builtin_fabsf(b));
}

// Scale byte of a block whose largest magnitude has the bits `top`.  448 is 1.75 * 2^8: adding 0x1fffff carries
// into the exponent exactly where the significand is above 1.75.
__device__ __forceinline__ unsigned scale8(unsigned top) {
  if (top >= kInf) return 255u;
  const int s = static_cast<int>((top + 0x1fffffu) >> 23) - 8;
  return s < 0 ? 0u : static_cast<unsigned>(s);
}
// 2^(s - 127); NaN for s = 255.
__device__ __forceinline__ float scale_value8(unsigned s) {
  return __builtin_bit_cast(float, s == 0 ? 0x00400000u : s == 255u ? 0x7fc00000u : s << 23);
}

// Four values of a block of scale byte s as four codes, each rounded once (to nearest, ties to even; what rounds to 2^128,
// the code 256 of the largest scale 247, goes to 240 there, so that finite values stay finite): the conversion
// divides by its scale operand's power of two (exponent 0 is 2^-127).  With it and the maximum of three above, a
// product of 65,536 x 4,096 x 1,024 into 8-bit rows takes 287 instead of 293 us, and with GELU 386 instead of 398.
__device__ __forceinline__ unsigned encode8(float a, float b, float c, float d, unsigned s) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  const float scale = __builtin_bit_cast(float, s << 23);
  i16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(i16x2{0, 0}, a, b, scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  unsigned codes = __builtin_bit_cast(unsigned, r);
  if (__builtin_amdgcn_ballot_w64(s >= 247u)) {  // a branch that few waves take
    const unsigned over = s == 247u ? ((codes & 0x7f7f7f7fu) + 0x08080808u) & 0x80808080u : 0u;  // 0x78 (256) is the only code past 0x77
    codes = s == 255u ? 0x7f7f7f7fu : codes - (over >> 7);
  }
  return codes;
}

// Largest magnitude bits over the 8 lanes of a 32-value block (4 values a lane, lanes 8 j .. 8 j + 7).
__device__ __forceinline__ unsigned block_top8(unsigned top) {
#pragma unroll
  for (int d = 1; d <= 4; d <<= 1) {
    const unsigned o = __shfl_xor(top, d, kWave);
    top = top > o ? top : o;
  }
  return top;
}

}  // namespace laya
