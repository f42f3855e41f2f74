// Matrix product of 8-bit rows: out = act(x w^T + bias) + residual, x [M][K] and w [N][K] in the form of rows8.hpp.
//
// Exact products: a code times its scale is a bf16 value (4 significant bits), so the codes are widened in
// registers, with their scales, by v_cvt_scalef32_pk_bf16_fp8 and multiplied by v_mfma_f32_16x16x32_bf16, whose sums
// are fp32 (measured: 8e-8 of the result's norm at K = 4,096).  It moves half the bytes of the 16-bit product, which is
// what few rows are bound by (1 x 4,096 x 1,024 4.9 us, 96 x 2,304 x 768 6.2, both a launch and one or two memory round
// trips; 512 x 1,024 x 4,096 with fp32 output 14.4, operand stream and widening).
// The 8-bit unit (kFast): v_mfma_scale_f32_16x16x128_f8f6f4 takes codes and scales as they are, at twice the rate, but
// aligns each 8 neighbouring products to their largest sum of exponents (a subnormal code's is its type's least) and cuts
// them off 2^13 below it, towards zero (measured with one large product and one small, normal and subnormal, and with
// significands of 1.125 to 1.875; the groups' sums are then added to 24 bits).
// Normal operands lose 2e-5 of the root of the products' sum of squares (1e-4 at most), where a channel in 128 is a
// thousand times the others and the products have one sign 1.6e-4 of their magnitudes (6e-4 at most): no sum in 32 bits. So
// a product takes it only where its caller says so, and never for fp32 outputs.
//
// Layout: whole 128-code slabs go straight from global memory into LDS, 16-byte chunk c of row r at position
// c ^ (r / 2) % 8, so that 16 lanes reading one chunk of 16 consecutive rows touch all banks once.  A workgroup
// owns BM x BN outputs, WM x WN waves of it times KG groups that split the slabs; S stages of SL slabs are in
// flight.  The groups' fp32 tiles are added in group order through LDS, so results do not depend on timing.
#include "kernels.hpp"
#include "linear8_plan.hpp"
#include "ring_walk.hpp"
#include "rows8.hpp"
#include "tiles.hpp"

#include <algorithm>
#include <type_traits>

namespace laya {

namespace {

// Direct loads as lds_load16_buffer, 16 bytes and 4 bytes a lane (lane l's go to LDS byte address lds + 16 l or 4 l), for
// resources that vector instructions may just have written (readfirstlane, the readlane of a spilled one): s_nop 4
// is the five wait states that such an SGPR needs before a vector-memory instruction reads it.
__device__ __forceinline__ void load_lds16(i32x4 rsrc, unsigned voffset, unsigned soffset, unsigned lds) {
  soffset = __builtin_amdgcn_readfirstlane(soffset);
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(lds));
}
__device__ __forceinline__ void load_lds4(i32x4 rsrc, unsigned voffset, unsigned soffset, unsigned lds) {
  soffset = __builtin_amdgcn_readfirstlane(soffset);
  asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(lds));
}

// Resource over `rows` rows of `pitch` bytes from row `first`: rows past the last read as zeros.
__device__ __forceinline__ i32x4 rows_resource(const uint8_t* base, long long first, long long rows, int limit, int pitch) {
  const long long n = rows - first < limit ? (rows > first ? rows - first : 0) : limit;
  return buffer_resource(base + (n > 0 ? first : 0) * pitch, static_cast<unsigned>(n * pitch));
}

// Eight codes (two dwords) times 2^(s - 127), `scale` holding s in a float's exponent: exact in bf16 (the hardware
// takes exponent 0 as 2^-127 and 255 as NaN; values under 2^-126 count as zero in the product).
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
// D = A(16x128) * B(128x16) + C of e4m3 codes with a scale per 32: lane l supplies row/column l % 16, its codes 16 (l / 16)
// .. +15 and 64 + 16 (l / 16) .. +15, and in the low byte of its scale that of codes 32 (l / 16) .. +31 of the row.
__device__ __forceinline__ f32x4 mfma8(i32x8 a, i32x8 b, f32x4 c, unsigned sa, unsigned sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// Activations, accurate to 3e-7 absolute (gelu16 with its argument capped where its tail has reached 0; SiLU by the
// hardware's exponential and reciprocal, a few units in the last place).  NaNs stay NaNs (the maximum is IEEE 754-2019's)
// and +infinity stays itself.
__device__ __forceinline__ float gelu8(float x) {
  const float ax = fminf(fabsf(x), 16.f);
  return __builtin_fmaf(-ax, gelu16_tail(ax), __builtin_elementwise_maximum(x, 0.f));
}
__device__ __forceinline__ float silu8(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

__host__ __device__ constexpr bool gated(Act8 act) { return act == Act8::Geglu || act == Act8::Swiglu; }

template <typename T> struct Vec { typedef T type __attribute__((ext_vector_type(4))); };

// Whole quad `at` of a tensor.
template <typename T>
__device__ __forceinline__ typename Vec<T>::type quad_at(const void* p, size_t at) {
  return *reinterpret_cast<const typename Vec<T>::type*>(static_cast<const T*>(p) + at);
}
// Residual columns n .. n + 3 of U places, zeros past the columns; every load goes out before the first is used.
template <int U>
__device__ __forceinline__ void load_residual(const Linear8Args& a, const long long (&row)[U], const int (&n)[U], const bool (&in)[U],
                                              float (&r)[U][4]) {
  auto load = [&](auto zero) {
    typedef decltype(zero) T;
    if (a.vec) {
      typename Vec<T>::type t[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (in[u] && n[u] < a.cols) t[u] = quad_at<T>(a.residual, static_cast<size_t>(row[u]) * a.cols + n[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) r[u][i] = in[u] && n[u] < a.cols ? static_cast<float>(t[u][i]) : 0.f;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          r[u][i] = in[u] && n[u] + i < a.cols ? static_cast<float>(static_cast<const T*>(a.residual)[static_cast<size_t>(row[u]) * a.cols + n[u] + i]) : 0.f;
    }
  };
  if (a.residual_type == static_cast<int>(DType::F32)) load(0.f);
  else if (a.residual_type == static_cast<int>(DType::F16)) load(f16());
  else load(bf16());
}
template <typename T>
__device__ __forceinline__ void store4(const Linear8Args& a, long long row, int n, const float (&v)[4]) {
  T* const dst = static_cast<T*>(a.out) + static_cast<size_t>(row) * a.cols + n;
  if (a.vec && n < a.cols) {
    *reinterpret_cast<typename Vec<T>::type*>(dst) =
        typename Vec<T>::type{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.cols) dst[i] = static_cast<T>(v[i]);
  }
}
// Two values as two 16-bit ones of `type`.
__device__ __forceinline__ unsigned pack16(int type, float x, float y) {
  if (type == static_cast<int>(DType::F16)) {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, f16x2{static_cast<f16>(x), static_cast<f16>(y)});
  }
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, bf16x2{static_cast<bf16>(x), static_cast<bf16>(y)});
}

// Columns n .. n + 3 of row `row` as codes: 8 lanes with consecutive quads of the same row (a whole block) all call;
// columns past `cols` come in as zeros and become the row's padding.
__device__ __forceinline__ void store_codes4(const Linear8Args& a, long long row, int n, const float (&v)[4]) {
  const unsigned s = scale8(block_top8(magnitude(largest(largest(0.f, v[0], v[1]), v[2], v[3]))));
  const size_t ld = static_cast<size_t>(padded8(a.cols));
  *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(a.out) + row * ld + n) = encode8(v[0], v[1], v[2], v[3], s);
  if (n % kBlock8 == 0) a.out_scales[row * (ld / kBlock8) + n / kBlock8] = static_cast<uint8_t>(s);
}

// Dwords of a slab's scales in LDS: x's rows, then w's, each in whole 64-row loads.
constexpr int scale_rows8(int rows) { return (rows + 63) / 64 * 64; }
template <int BM, int BN, int SL> constexpr int stage_bytes8() {
  return SL * ((BM + BN) * 128 + (scale_rows8(BM) + scale_rows8(BN)) * 4);
}
template <int BM, int BN, int KG, int SL, int S> constexpr int lds8() {
  const int stages = S * stage_bytes8<BM, BN, SL>(), parts = KG * BM * (BN + 4) * 4;
  return (stages > parts ? stages : parts) + BN * 4;  // and the tile's bias
}

// Waves a SIMD: two workgroups a CU where their LDS fits.
template <int NT> constexpr int waves8(int lds) { return (2 * lds <= 160 * 1024 ? 2 : 1) * NT / 256; }

template <int BM, int BN, int WM, int WN, int KG, int SL, int S, bool kFast>
__global__ __launch_bounds__(64 * WM * WN * KG, waves8<64 * WM * WN * KG>(lds8<BM, BN, KG, SL, S>())) void linear8_kernel(Linear8Args a) {
  constexpr int NW = WM * WN * KG, NT = 64 * NW;
  constexpr int WTM = BM / WM, WTN = BN / WN, MB = WTM / 16, NB = WTN / 16;
  static_assert(MB >= 1 && NB >= 1 && WTM % 16 == 0 && WTN % 16 == 0, "16x16 MFMA blocks");
  constexpr int PITCH = BN + 4;  // floats per row of a partial tile: 16-byte rows, spread over the banks
  constexpr int RG = (BM + BN) / 8, SX = scale_rows8(BM), SG = (SX + scale_rows8(BN)) / 64;
  constexpr int STAGE = stage_bytes8<BM, BN, SL>(), CODES = SL * (BM + BN) * 128;
  constexpr int GROUPS = SL * (RG + SG);
  constexpr int NLD = (GROUPS + NW - 1) / NW;  // loads per wave and stage; past the last, the last again
  static_assert((S - 1) * NLD < 64 && lds8<BM, BN, KG, SL, S>() <= 160 * 1024, "vmcnt range and LDS of a CU");
  extern __shared__ __align__(16) unsigned char smem_raw[];
  float* const red = reinterpret_cast<float*>(smem_raw);  // [KG][BM][PITCH], after the main loop
  float* const sbias = reinterpret_cast<float*>(smem_raw + lds8<BM, BN, KG, SL, S>() - BN * 4);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool glu = gated(a.act);
  const int oc = glu ? BN / 2 : BN;  // output columns of a tile
  const int span = a.out_type == kE4M3 ? static_cast<int>(padded8(a.cols)) : a.cols;
  int tx, ty, tz;
  tile_of_even(blockIdx.x, (span + oc - 1) / oc, (a.M + BM - 1) / BM, 1, &tx, &ty, &tz);
  const long long n0 = static_cast<long long>(tx) * BN, m0 = static_cast<long long>(ty) * BM;

  const int sld = a.ld / kBlock8;  // scale bytes of a row
  const i32x4 rsX = rows_resource(a.x, m0, a.M, BM, a.ld), rsXs = rows_resource(a.xs, m0, a.M, BM, sld);
  const i32x4 rsW = rows_resource(a.w, n0, a.N, BN, a.ld), rsWs = rows_resource(a.ws, n0, a.N, BN, sld);
  const bool live = n0 < a.N;
  const unsigned lds_base = lds_address(smem_raw);
  const int n = a.ld / 128, stages = (n + SL - 1) / SL;

  // Load group g of a stage: the SL slabs' 8-row code groups, then their 64-row scale groups (a dword of four
  // scales per row and slab); x's rows before w's.
  auto issue = [&](int stage, int buf) {
#pragma unroll
    for (int q = 0; q < NLD; ++q) {
      const int g = min(wave + NW * q, GROUPS - 1);
      const unsigned base = lds_base + static_cast<unsigned>(buf * STAGE);
      if (g < SL * RG) {
        const int rg = g % RG, r = rg * 8 + (lane >> 3);
        const unsigned k = static_cast<unsigned>(min(stage * SL + g / RG, n - 1)) * 128u;
        const bool isx = rg * 8 < BM;  // a scalar offset has to stay inside its resource: 0 where w has no rows
        const unsigned row = static_cast<unsigned>(isx ? r : r - BM);
        load_lds16(isx ? rsX : rsW, row * static_cast<unsigned>(a.ld) + (((lane & 7) ^ ((r >> 1) & 7)) << 4),
                          isx || live ? k : 0u,
                          base + static_cast<unsigned>(g * 1024));
      } else {
        const int sg = (g - SL * RG) % SG, r = sg * 64 + lane;
        const unsigned k = static_cast<unsigned>(min(stage * SL + (g - SL * RG) / SG, n - 1)) * 4u;
        const bool isx = sg * 64 < SX;
        const unsigned row = static_cast<unsigned>(isx ? r : r - SX);
        load_lds4(isx ? rsXs : rsWs, row * static_cast<unsigned>(sld), isx || live ? k : 0u,
                         base + static_cast<unsigned>(CODES + (g - SL * RG) * 256));
      }
    }
  };

  static_assert(NT >= BN, "a thread per bias column");
  const float early_bias = a.bias && tid < BN && n0 + tid < a.N ? a.bias[n0 + tid] : 0.f;

  const int kg = wave / (WM * WN), wm0 = (wave % (WM * WN)) / WN * WTM, wn0 = wave % WN * WTN;
  const int r16 = lane & 15, kq = lane >> 4;
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](int buf, int count) {
    constexpr int PS = (SL + KG - 1) / KG;
#pragma unroll
    for (int u = 0; u < PS; ++u) {
      const int slab = kg + u * KG;
      if (slab < count) {
        const unsigned char* const codes = smem_raw + buf * STAGE + slab * (BM + BN) * 128;
        const unsigned* const sc = reinterpret_cast<const unsigned*>(smem_raw + buf * STAGE + CODES) + slab * SG * 64;
        // Lane group kq takes the 16 codes at 16 kq of each half of the slab.
        auto chunk = [&](int r, int h) {
          return *reinterpret_cast<const i32x4*>(codes + r * 128 + (((4 * h + kq) ^ ((r >> 1) & 7)) << 4));
        };
        unsigned sx[MB], sw[NB];
        if constexpr (kFast) {
          // One MFMA per slab and 16x16 block: the instruction takes the scale of its lane's own 32 codes in k order,
          // block kq of the row.
#pragma unroll
          for (int i = 0; i < MB; ++i) sx[i] = sc[wm0 + i * 16 + r16] >> (8 * kq);
#pragma unroll
          for (int j = 0; j < NB; ++j) sw[j] = sc[SX + wn0 + j * 16 + r16] >> (8 * kq);
          i32x8 fx[MB], fw[NB];
          auto fragment = [&](int r) {
            const i32x4 lo = chunk(r, 0), hi = chunk(r, 1);
            return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          };
#pragma unroll
          for (int i = 0; i < MB; ++i) fx[i] = fragment(wm0 + i * 16 + r16);
#pragma unroll
          for (int j = 0; j < NB; ++j) fw[j] = fragment(BM + wn0 + j * 16 + r16);
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = mfma8(fw[j], fx[i], acc[i][j], sw[j], sx[i]);
        } else {
          // Each half's 16 codes lie in block kq / 2 of it: two bf16 operands of 8 (any order of k will do that x
          // and w share).
#pragma unroll
          for (int i = 0; i < MB; ++i) sx[i] = sc[wm0 + i * 16 + r16] >> (8 * (kq >> 1));
#pragma unroll
          for (int j = 0; j < NB; ++j) sw[j] = sc[SX + wn0 + j * 16 + r16] >> (8 * (kq >> 1));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            auto fragment = [&](int r, unsigned s, bf16x8 (&f)[2]) {
              const i32x4 c = chunk(r, h);
              const float scale = __builtin_bit_cast(float, ((s >> (16 * h)) & 255u) << 23);
              f[0] = widen8(c[0], c[1], scale);
              f[1] = widen8(c[2], c[3], scale);
            };
            bf16x8 fx[MB][2], fw[NB][2];
#pragma unroll
            for (int i = 0; i < MB; ++i) fragment(wm0 + i * 16 + r16, sx[i], fx[i]);
#pragma unroll
            for (int j = 0; j < NB; ++j) fragment(BM + wn0 + j * 16 + r16, sw[j], fw[j]);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = mfma16(fw[j][e], fx[i][e], acc[i][j]);
          }
        }
      }
    }
  };

  // Every stage's barrier makes its loads visible and ends the reads of the stage before it, whose buffer then
  // takes stage it + S - 1.
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < stages) issue(s, s);
  int buf = 0;
  for (int it = 0; it < stages; ++it) {
    const int younger = min(it ? S - 2 : S - 1, stages - 1 - it);  // stages in flight behind this one
    if (S >= 4 && younger >= 3) publish_stage<waitcnt_vm(S >= 4 ? 3 * NLD : 0)>();
    else if (S >= 3 && younger >= 2) publish_stage<waitcnt_vm(S >= 3 ? 2 * NLD : 0)>();
    else if (S >= 2 && younger >= 1) publish_stage<waitcnt_vm(NLD)>();
    else publish_stage<waitcnt_vm(0)>();
    if (it && it + S - 1 < stages) issue(it + S - 1, buf ? buf - 1 : S - 1);
    compute(buf, min(SL, n - it * SL));
    buf = buf + 1 == S ? 0 : buf + 1;
  }
  __syncthreads();  // the partial tiles reuse the stages

  if (tid < BN) sbias[tid] = early_bias;
  float* const mine = red + kg * BM * PITCH;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      *reinterpret_cast<f32x4*>(mine + (wm0 + i * 16 + r16) * PITCH + wn0 + j * 16 + 4 * kq) = acc[i][j];
  __syncthreads();

  // Four columns n .. n + 3 of tile row r: the groups' sum in group order, and the bias (zeros past N).
  auto total4 = [&](int r, int n, float (&v)[4]) {
    f32x4 t = *reinterpret_cast<const f32x4*>(red + r * PITCH + n);
#pragma unroll
    for (int w = 1; w < KG; ++w) {
      const f32x4 o = *reinterpret_cast<const f32x4*>(red + (w * BM + r) * PITCH + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = t[e] + o[e];
    }
    const f32x4 b = *reinterpret_cast<const f32x4*>(sbias + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = t[e] + b[e];
  };
  // A thread's quads go U at a time through each step, so that their LDS reads, their residual's loads and their
  // activations overlap: against one at a time 2,000 x 1,024 x 4,096 with a residual 23.7 -> 22.8 us, 300 x 2,304 x 768 6.1 ->
  // 5.9.  Two where 128 registers are all that a wave has (128 x 128 tiles, two workgroups a CU: four spilled).
  constexpr int kMost = waves8<NT>(lds8<BM, BN, KG, SL, S>()) >= 4 ? 2 : 4;
  auto write = [&](auto glu_c) {
    constexpr bool kGlu = decltype(glu_c)::value;
    constexpr int OC = kGlu ? BN / 2 : BN, Q = OC / 4, QUADS = (BM * Q + NT - 1) / NT, U = QUADS < kMost ? QUADS : kMost;
    static_assert(QUADS % U == 0, "whole steps");
    int first = tid;
    if constexpr (QUADS >= 8) asm volatile("" : "+v"(first));  // opaque: the addresses stay out of the main loop's registers
#pragma unroll 1
    for (int c0 = first; c0 < BM * Q; c0 += U * NT) {
      float v[U][4], res[U][4];
      long long row[U];
      int col[U];
      bool in[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * NT, r = c / Q;
        row[u] = m0 + r;
        col[u] = tx * OC + (c % Q) * 4;
        in[u] = c < BM * Q && row[u] < a.M && col[u] < span;  // alike in the 8 lanes of a block
      }
      if (a.residual) load_residual(a, row, col, in, res);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = min(c0 + u * NT, BM * Q - 1), r = c / Q, f = (c % Q) * 4;
        if constexpr (kGlu) {
          float g[4];
          const int n = (f / 16) * 32 + f % 16;
          total4(r, n, g);
          total4(r, n + 16, v[u]);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = (a.act == Act8::Geglu ? gelu8(g[e]) : silu8(g[e])) * v[u][e];
        } else {
          total4(r, f, v[u]);
        }
      }
      if (!kGlu && a.act == Act8::Gelu) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = gelu8(v[u][e]);
      } else if (!kGlu && a.act == Act8::Relu) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = v[u][e] < 0.f ? 0.f : v[u][e];
      }
      if (a.residual) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = v[u][e] + res[u][e];
      }
      auto store = [&](auto one) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (in[u]) one(u);
      };
      if (a.out_type == kE4M3) store([&](int u) { store_codes4(a, row[u], col[u], v[u]); });
      else if (a.out_type == static_cast<int>(DType::F32)) store([&](int u) { store4<float>(a, row[u], col[u], v[u]); });
      else if (a.out_type == static_cast<int>(DType::F16)) store([&](int u) { store4<f16>(a, row[u], col[u], v[u]); });
      else store([&](int u) { store4<bf16>(a, row[u], col[u], v[u]); });
    }
  };
  if constexpr (BN % 32 == 0) {
    if (glu) return write(std::true_type());
  }
  write(std::false_type());
}

// ---- the batched product: a persistent ring of 256 x 256 tiles ----

constexpr int kUnit8 = 64 * 128;   // bytes of a ring unit: 64 rows of one slab
constexpr int kSlab8 = 8 * kUnit8;  // four units of x, four of w
constexpr int kScaleStages8 = 3;
constexpr int kScales8 = 2 * kSlab8, kScaleStage8 = 512 * 4;
constexpr int kBias8 = kScales8 + kScaleStages8 * kScaleStage8;  // two tiles' bias, 256 floats each
constexpr int kRing8Lds = kBias8 + 2 * 1024;
static_assert(kRing8Lds <= 160 * 1024, "LDS of a CU");

// Exchanges between the four lane groups (lanes 16 q .. 16 q + 15).
// v[j] of group q: afterwards v[k] of group j holds what was v[j] of group k.
__device__ __forceinline__ void transpose4(unsigned (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const auto r = __builtin_amdgcn_permlane32_swap(v[j], v[j + 2], false, false);
    v[j] = r[0];
    v[j + 2] = r[1];
  }
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(v[j], v[j + 1], false, false);
    v[j] = r[0];
    v[j + 1] = r[1];
  }
}
// x and y of group q are chunks q of two runs of four: afterwards groups 0 and 1 hold x's chunks (0, 1) and (2, 3) in x and
// y, groups 2 and 3 y's.
__device__ __forceinline__ void pair_chunks(unsigned& x, unsigned& y) {
  const auto a = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(a[0], a[1], false, false);
  x = b[0];
  y = b[1];
}
// Maximum over the four lane groups.
__device__ __forceinline__ unsigned group_max(unsigned m) {
  const auto a = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = a[0] > a[1] ? a[0] : a[1];
  const auto b = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return b[0] > b[1] ? b[0] : b[1];
}

// Eight waves on a 2 x 4 grid of 128 x 64 outputs; a grid of at most one workgroup per CU walks the tiles, and the
// operand stream runs on across tile boundaries.  LDS holds two slabs as units of 64 rows x 128 codes (of each of
// which every wave loads 8 rows) and three stages of scales.  A wave's slab is eight rows of four MFMAs (a 16-row
// block of x against its four 16-column blocks of w): w's fragments stay in registers for the slab, x's go through
// four register sets, read two rows ahead.  Two barriers a slab, each some rows after the reads it waits for:
//   before row 2: w's units and the first half of x's have been read and take the slab after the next;
//   before row 6: the second half of x's; the next slab's first fragments are read under rows 6 and 7.
// What a barrier publishes was issued three barriers earlier, one and a half slabs: with one barrier a slab (one
// slab for most loads) the loads' latency bounded the loop.
//
// The epilogue needs no LDS: lane (r, kq) = (lane % 16, lane / 16) holds columns 4 kq .. +3 of row r of each 16 x 16
// block, and the four lane groups exchange packed dwords so that each stores 16 bytes of consecutive columns.
//
// Exact products (kExact) take the same walk and stream: a slab is two passes, one per 64-code half,
// over the eight row blocks, with w's half widened for the pass and x's next row block widened between the MFMAs of
// the present one.  Its MFMAs take twice as long, so a barrier frees all of x's units, another all of w's.
//
// Measured, us by the card's clock: 65,536 x 1,024 x 4,096 on the 8-bit unit into bf16 262-320 (2.1-1.7 PFLOP/s); exact into
// bf16 430-455, fp32 445-460, with an fp32 residual 480-545.  65,536 x 4,096 x 1,024 on the unit into bf16 305-335, 8-bit rows
// 280-287, with GELU 343-386; exact 465-475, 450-465, 510-549.  The unit's MFMAs alone take 145 us, operand loads alone
// 202 (K = 4,096) and 109 (K = 1,024); a row of its MFMAs under which loads go out takes 1.5 to 1.9 times as long, and the
// epilogue 8,200 clocks a tile, 17,400 with GELU into 8-bit rows.
enum class Out8 { Half, E4m3, F32 };
template <Act8 A, Out8 O, bool kExact, bool kResidual>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void linear8_ring_kernel(Linear8Args a, RingWalk walk) {
  constexpr bool kGlu = gated(A), kE4m3 = O == Out8::E4m3, kF32 = O == Out8::F32;
  static_assert(kExact || !kF32, "fp32 outputs are made from exact products");
  constexpr int BM = 256, BN = 256, MB = 8, NB = 4;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;  // 128 rows, 64 columns
  const int r16 = lane & 15, kq = lane >> 4;

  const int span = kE4m3 ? static_cast<int>(padded8(a.cols)) : a.cols;
  const int total = walk.total, G = gridDim.x;
  const int n = a.ld / 128;  // slabs of a tile (the launcher checks n >= 2)
  const int sld = a.ld / kBlock8;
  int id = blockIdx.x;
  if (id >= total) return;

  struct Tile {
    int m0, n0;
    i32x4 x, w, s;  // codes, and the scales of this wave's load
    bool live;      // holds rows of w (a tile of an 8-bit output's padding need not)
  };
  auto open = [&](int t) {
    int tx, ty;
    ring_tile(walk, t, &tx, &ty);
    Tile k;
    k.m0 = ty * BM;
    k.n0 = tx * BN;
    const int mr = max(min(a.M - k.m0, BM), 0), nr = max(min(a.N - k.n0, BN), 0), nf = min(k.n0, a.N);
    k.live = nr > 0;
    k.x = buffer_resource(a.x + static_cast<size_t>(k.m0) * a.ld, mr * a.ld);
    k.w = buffer_resource(a.w + static_cast<size_t>(nf) * a.ld, nr * a.ld);
    k.s = wave < 4 ? buffer_resource(a.xs + static_cast<size_t>(k.m0) * sld, mr * sld)
                   : buffer_resource(a.ws + static_cast<size_t>(nf) * sld, nr * sld);
    return k;
  };
  Tile cur = open(id), nxt = cur;
  int nid = id + G;
  bool has_next = nid < total;
  if (has_next) nxt = open(nid);

  const unsigned lds_base = lds_address(smem_raw);
  unsigned src[4];  // byte offset of this lane's 16 codes in each 64-row unit of an operand
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = u * 64 + wave * 8 + (lane >> 3);
    src[u] = static_cast<unsigned>(r) * static_cast<unsigned>(a.ld) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
  }
  // Scales of 64 rows: dword 4 r + j of the load is row 16 j + r, so that a lane reads those of its row of four
  // 16-row blocks at once.
  const unsigned src_scale = static_cast<unsigned>((wave & 3) * 64 + (lane & 3) * 16 + (lane >> 2)) * static_cast<unsigned>(sld);

  // A scalar offset has to stay inside its resource (ranges.hpp): where w has no rows it is 0, and the loads read zeros.
  // Loads of stream slab `s` counted from this tile's first: this tile's, the next one's, or (last tile) this
  // tile's last again, never read.
  auto issue = [&](int u, int s, int buf) {
    const bool next = s >= n && has_next;
    const int kt = (u < 4 || (next ? nxt.live : cur.live)) ? (next ? s - n : min(s, n - 1)) : 0;
    load_lds16(u < 4 ? (next ? nxt.x : cur.x) : (next ? nxt.w : cur.w), src[u & 3], static_cast<unsigned>(kt) * 128u,
                      lds_base + static_cast<unsigned>(buf * kSlab8 + u * kUnit8 + wave * 1024));
  };
  auto issue_scales = [&](int s, int stage) {
    const bool next = s >= n && has_next;
    const int kt = (wave < 4 || (next ? nxt.live : cur.live)) ? (next ? s - n : min(s, n - 1)) : 0;
    load_lds4(next ? nxt.s : cur.s, src_scale, static_cast<unsigned>(kt) * 4u,
                     lds_base + static_cast<unsigned>(kScales8 + stage * kScaleStage8 + wave * 256));
  };

  // Fragment addresses: a lane's two chunks, kq and 4 + kq, lie 64 bytes apart under the swizzle of its row.
  const int frag = r16 * 128 + ((kq ^ (r16 >> 1)) << 4);
  i32x8 fx[4], fw[NB];
  unsigned sx[MB], sw[NB];
  // A slab's addresses: one register pair per operand, the blocks at constant offsets from it.  Opaque to the compiler,
  // which kept a pair per buffer and block otherwise, and spilled.
  struct Place {
    int lo, hi;
  };
  auto place = [&](int base) {
    Place p{base + frag, (base + frag) ^ 64};
    asm volatile("" : "+v"(p.lo), "+v"(p.hi));
    return p;
  };
  auto read = [&](const Place& p, int offset) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(smem_raw + p.lo + offset);
    const i32x4 hi = *reinterpret_cast<const i32x4*>(smem_raw + p.hi + offset);
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto place_x = [&](int buf) { return place(buf * kSlab8 + wm * 2 * kUnit8); };
  auto place_w = [&](int buf) { return place(buf * kSlab8 + (4 + wn) * kUnit8); };
  auto read_x = [&](const Place& p, int i) { fx[i & 3] = read(p, i * 2048); };
  auto read_w = [&](const Place& p, int j) { fw[j] = read(p, j * 2048); };
  // Scale dwords of four 16-row blocks; `settle` moves the byte of the lane's 32 codes down.  It comes two rows after
  // the read: the schedule's pins keep it where it is written, and it waits for the read.
  auto read_scales = [&](int stage, int group, unsigned* s) {
    const i32x4 v = *reinterpret_cast<const i32x4*>(smem_raw + kScales8 + stage * kScaleStage8 + group * 256 + r16 * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = static_cast<unsigned>(v[j]);
  };
  auto settle = [&](unsigned* s, const unsigned* raw) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = raw[j] >> (8 * kq);
  };
  f32x4 acc[MB][NB];
  auto mma = [&](int i, int j) {  // weights as the MFMA's A operand: the accumulator holds C^T
    acc[i][j] = mfma8(fw[j], fx[i & 3], acc[i][j], sw[j], sx[i]);
    // Emits nothing; as MFMAs have no side effects, the compiler moved them past barriers, holding all their fragments.
    asm volatile("" : "+v"(acc[i][j]));
  };
  auto pin = [] { __builtin_amdgcn_sched_barrier(0); };

  // The tile's bias, zeros past N, into its half of the bias area (every wave loads 64 columns, twice over).
  auto issue_bias = [&](int half) {
    const int nr = a.bias ? max(min(a.N - cur.n0, BN), 0) : 0;
    load_lds4(buffer_resource(a.bias + (nr ? cur.n0 : 0), nr * 4), static_cast<unsigned>((wave & 3) * 256 + lane * 4), 0,
                     lds_base + static_cast<unsigned>(kBias8 + half * 1024 + (wave & 3) * 256));
  };
  issue_bias(0);
  // Of the two waves of a SIMD the second goes first where both could: apart, one's MFMAs cover the other's reads (up to
  // 2% of a batched product, 4% of a one-round one).
  if (wm) __builtin_amdgcn_s_setprio(1);

  // The two groups of a slab's loads, and what each barrier leaves in flight beside the stores (below).
  // Before row 2: scales, w and the first half of x; before row 6: the rest of x.  kExact: scales and w; x.
  auto issue_first = [&](int part, int s, int buf, int stage) {
    if (part == 0) issue_scales(s, stage);
    issue(4 + part, s, buf);
    if (!kExact && (part == 1 || part == 2)) issue(part == 1 ? 0 : 2, s, buf);
  };
  auto issue_second = [&](int part, int s, int buf) {
    issue(kExact ? 2 * part : 2 * part + 1, s, buf);
    if (kExact) issue(2 * part + 1, s, buf);
  };
  constexpr int kFirst = kExact ? 5 : 7, kSecond = 9 - kFirst;

  // Prologue: slabs 0 and 1.
  int buf = 0, stage = 0, half = 0;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int q = 0; q < 4; ++q) issue_first(q, s, s, s);
    issue_second(0, s, s);
    issue_second(1, s, s);
  }
  publish_stage<waitcnt_vm(0)>();  // both slabs: the first tile's first slab waits as the later tiles' do
  auto next_stage = [](int s) { return s == kScaleStages8 - 1 ? 0 : s + 1; };

  // kExact: a lane's half (h) of a 16-row block is 16 codes of block kq / 2 of the half, two bf16 operands of 8.
  i32x4 cx[4], cw[NB], xa[2], xb[2];
  bf16x8 ww[NB][2];
  auto read_cx = [&](const Place& p, int h, int i) {
    cx[i & 3] = *reinterpret_cast<const i32x4*>(smem_raw + (h ? p.hi : p.lo) + i * 2048);
  };
  auto read_cw = [&](const Place& p, int h, int j) {
    cw[j] = *reinterpret_cast<const i32x4*>(smem_raw + (h ? p.hi : p.lo) + j * 2048);
  };
  auto half_scale = [&](unsigned s, int h) {
    return __builtin_bit_cast(float, ((s >> (8 * (kq >> 1) + 16 * h)) & 255u) << 23);
  };
  auto widen_w = [&](int h, int j) {
    const float f = half_scale(sw[j], h);
    ww[j][0] = widen8(cw[j][0], cw[j][1], f);
    ww[j][1] = widen8(cw[j][2], cw[j][3], f);
  };
  // Two of the 16 codes of x's row block i into xb.
  auto widen_x = [&](float f, int i, int k) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const int c = cx[i & 3][k >> 1];
    const bf16x2 v = k & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, f, false);
    int d = __builtin_bit_cast(int, v);
    asm volatile("" : "+v"(d));  // stays between the MFMAs
    xb[k >> 2][k & 3] = d;
  };
  auto mma_exact = [&](int i, int j, int e) {
    acc[i][j] = mfma16(ww[j][e], __builtin_bit_cast(bf16x8, xa[e]), acc[i][j]);
    asm volatile("" : "+v"(acc[i][j]));
  };

  // What rows 0 and 1 of a slab need.
  auto read_first = [&] {
    if constexpr (kExact) {
      read_scales(stage, 2 * wm, sx);
      read_scales(stage, 2 * wm + 1, sx + 4);
      read_scales(stage, 4 + wn, sw);
      const Place px = place_x(buf), pw = place_w(buf);
#pragma unroll
      for (int j = 0; j < NB; ++j) read_cw(pw, 0, j);
#pragma unroll
      for (int i = 0; i < 3; ++i) read_cx(px, 0, i);
#pragma unroll
      for (int j = 0; j < NB; ++j) widen_w(0, j);
      const float f = half_scale(sx[0], 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) widen_x(f, 0, k);
      xa[0] = xb[0];
      xa[1] = xb[1];
      return;
    }
    read_scales(stage, 2 * wm, sx);
    read_scales(stage, 4 + wn, sw);
    const Place px = place_x(buf), pw = place_w(buf);
    read_x(px, 0);
#pragma unroll
    for (int j = 0; j < NB; ++j) read_w(pw, j);
    read_x(px, 1);
    settle(sx, sx);
    settle(sw, sw);
  };
  read_first();

  // The waits leave what is younger than the loads that the barrier publishes in flight: a group of each kind, and in a
  // tile's first slab (kLate) the epilogue stores and the bias load, which come between the two tiles' loads.  Waiting
  // for the stores there cost 2-3 us a tile.  (No wait is chosen at run time: across the branch the compiler moved
  // the MFMAs behind the barrier.)
  constexpr int kStores = (kGlu ? MB : 2 * MB) * (kF32 ? 2 : 1);
  constexpr int kWait = kExact ? kFirst : kFirst + kSecond, kWaitLate = kWait + kStores + 1;
  auto four = [&](int i) {
    pin();
#pragma unroll
    for (int j = 0; j < NB; ++j) mma(i, j);
    pin();
  };
  // Rows 0 .. 5 of the slab in `buf`; `to`: the stream slab whose loads go out.
  auto first_rows = [&](int to, auto late) {
    constexpr int kVm = decltype(late)::value ? kWaitLate : kWait;
    const int tostage = next_stage(next_stage(stage));
    const Place px = place_x(buf);
    read_x(px, 2);
    four(0);
    read_scales(stage, 2 * wm + 1, sx + 4);
    read_x(px, 3);
    four(1);
    publish_stage<waitcnt_vm(kVm)>();
    pin();
#pragma unroll
    for (int i = 2; i < 6; ++i) {
      issue_first(i - 2, to, buf, tostage);
      if (i == 3) settle(sx + 4, sx + 4);
      read_x(px, i + 2);
      four(i);
    }
    publish_stage<waitcnt_vm(kVm)>();
    pin();
  };
  // Rows 6 and 7, column by column, so that each of w's fragments is free for the next slab's (kNext) early.
  auto last_rows = [&](int to, auto next) {
    constexpr bool kNext = decltype(next)::value;
    const int nstage = next_stage(stage);
    unsigned nw[4];
    if constexpr (kNext) {
      read_scales(nstage, 2 * wm, sx);
      read_scales(nstage, 4 + wn, nw);
    }
    const Place px = place_x(buf ^ 1), pw = place_w(buf ^ 1);
    if constexpr (kNext) read_x(px, 0);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (j == 0) issue_second(0, to, buf);
      if (j == 2) issue_second(1, to, buf);
      pin();
      mma(6, j);
      mma(7, j);
      pin();
      if constexpr (kNext) {
        read_w(pw, j);
        if (j == 1) read_x(px, 1);
        if (j == 2) settle(sx, sx);
        if (j == 3) settle(sw, nw);
      }
    }
    buf ^= 1;
    stage = nstage;
  };

  // kExact: a slab, its row blocks numbered t = 8 h + i.  Row block t + 1 is widened under t's MFMAs, t + 3 read; at
  // the end of a pass w's next half is widened column by column as its registers come free.
  auto exact_slab = [&](int to, auto late, auto next) {
    constexpr bool kNext = decltype(next)::value;
    constexpr int kVm = decltype(late)::value ? kWaitLate : kWait;
    const int nstage = next_stage(stage), tostage = next_stage(nstage);
    const Place px = place_x(buf), pw = place_w(buf);
    Place qx = px;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const int i = t & 7, u = t + 1;
      if (t == 3) {  // w has been read
        __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0_keep_vm());
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        pin();
      }
      if (t == 13) {  // x has been read, and the next slab is there
        publish_stage<waitcnt_vm(kVm)>();
        pin();
        if constexpr (kNext) {
          qx = place_x(buf ^ 1);
          const Place qw = place_w(buf ^ 1);
          read_scales(nstage, 2 * wm, sx);
          read_scales(nstage, 4 + wn, sw);
#pragma unroll
          for (int j = 0; j < NB; ++j) read_cw(qw, 0, j);
        }
      }
      if (t >= 3 && t < 7) issue_first(t - 3, to, buf, tostage);
      if (t == 13 || t == 14) issue_second(t - 13, to, buf);
      if (t == 0) read_scales(stage, 2 * wm + 1, sx + 4);
      if (t < 2) {
        read_cw(pw, 1, 2 * t);
        read_cw(pw, 1, 2 * t + 1);
      }
      if (t < 13) read_cx(px, (t + 3) >> 3, (t + 3) & 7);
      else if (kNext) read_cx(qx, 0, t - 13);
      pin();
      const bool more = t < 15 || kNext;
      const float f = more ? half_scale(sx[u & 7], (u >> 3) & 1) : 0.f;
      if (i < 7) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          mma_exact(i, k & 3, k >> 2);
          widen_x(f, u & 7, k);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          mma_exact(i, j, 0);
          if (more) widen_x(f, u & 7, 2 * j);
          mma_exact(i, j, 1);
          if (more) widen_x(f, u & 7, 2 * j + 1);
          if (more) widen_w((u >> 3) & 1, j);
        }
      }
      pin();
      xa[0] = xb[0];
      xa[1] = xb[1];
    }
    buf ^= 1;
    stage = nstage;
  };

  for (;;) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (kExact) {
      exact_slab(2, std::true_type(), std::true_type());
      for (int it = 1; it < n - 1; ++it) exact_slab(it + 2, std::false_type(), std::true_type());
      exact_slab(n + 1, std::false_type(), std::false_type());
    } else {
      first_rows(2, std::true_type());
      for (int it = 1; it < n; ++it) {
        last_rows(it + 1, std::true_type());
        first_rows(it + 2, std::false_type());
      }
      // The tile's last slab: the next tile's first fragments are read after the epilogue.
      last_rows(n + 1, std::false_type());
    }

    // Epilogue, four 16 x 16 output blocks at a time: block t is a row block of the wave and its column block t
    // (gated: a pair of row blocks with two column blocks each).  Stores go through a resource over the tile's rows:
    // rows past M and columns past the row's end are dropped, and every wave issues the same number of them.
    int elane = lane;  // an opaque copy: the epilogue's addresses stay out of the main loop's registers
    asm volatile("" : "+v"(elane));
    const int er = elane & 15, eq = elane >> 4;
    constexpr int STEPS = kGlu ? MB / 2 : MB;
    constexpr unsigned kNowhere = 0x80000000u;  // past every resource
    // 8-bit codes past the caches (nontemporal): with the down projection behind it an FFN of 65,536 x 4,096 x 1,024 on the 8-bit
    // unit takes 716 instead of 723 us, of 4,096 rows 69.8 and 70.4, with exact products the same; other types lost by it.
    constexpr int kStream = kE4m3 ? 2 : 0;
    const int col0 = (kGlu ? cur.n0 / 2 + wn * 32 : cur.n0 + wn * 64);
    const int rows = min(a.M - cur.m0, BM);
    const int pitch = kE4m3 ? span : a.cols * (kF32 ? 4 : 2);  // bytes of an output row
    const __amdgpu_buffer_rsrc_t dst = __builtin_amdgcn_make_buffer_rsrc(
        static_cast<uint8_t*>(a.out) + static_cast<size_t>(cur.m0) * pitch, 0, rows * pitch, 0x00020000);
    const __amdgpu_buffer_rsrc_t dst_scales = __builtin_amdgcn_make_buffer_rsrc(
        kE4m3 ? a.out_scales + static_cast<size_t>(cur.m0) * (span / kBlock8) : nullptr, 0, kE4m3 ? rows * (span / kBlock8) : 0,
        0x00020000);
    const float* const bias = reinterpret_cast<const float*>(smem_raw + kBias8 + half * 1024) + wn * 64 + 4 * eq;
    // Row in the tile and first column of block t of a step.
    auto row_of = [&](int step, int t) { return wm * 128 + (kGlu ? 2 * step + (t >> 1) : step) * 16 + er; };
    auto block_col = [&](int t) { return col0 + (kGlu ? t & 1 : t) * 16; };
    // The residual's quads of a step, as they lie in memory (16-bit ones in the low half): all four loads go out before the
    // first is used (bf16 to bf16, 15,088 x 1,024 x 1,024 32.4 -> 28.3 us against one at a time, 65,536 x 1,024 x 4,096 307 -> 295;
    // fp32 551 -> 545, where the tile ends of all CUs meet at HBM).  The last of them waits for the step before's stores too, as
    // both share one in-order counter.  These kernels spill: 10 to 15 registers with exact products, 1 on the unit ungated; a step's
    // loads a whole step earlier spilled 55 and more.
    const int rsize = a.residual_type == static_cast<int>(DType::F32) ? 4 : 2;
    auto fetch_residual = [&](int step, u32x4 (&to)[4]) {
      pin();
      const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(static_cast<const uint8_t*>(a.residual)) + static_cast<size_t>(cur.m0) * a.cols * rsize, 0,
          rows * a.cols * rsize, 0x00020000);
      unsigned at[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int col = block_col(t) + 4 * eq;
        at[t] = col < a.cols ? static_cast<unsigned>((row_of(step, t) * a.cols + col) * rsize) : kNowhere;
      }
      if (rsize == 4) {
#pragma unroll
        for (int t = 0; t < 4; ++t) to[t] = __builtin_amdgcn_raw_buffer_load_b128(src, at[t], 0, 0);
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const auto q = __builtin_amdgcn_raw_buffer_load_b64(src, at[t], 0, 0);
          to[t][0] = q[0];
          to[t][1] = q[1];
        }
      }
    };
    auto add_residual = [&](const u32x4 (&from)[4], float (&v)[4][4]) {
      auto add = [&](auto zero) {
        typedef typename Vec<decltype(zero)>::type Q;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          Q q;
          __builtin_memcpy(&q, &from[t], sizeof(Q));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[t][e] = v[t][e] + static_cast<float>(q[e]);
        }
      };
      if (rsize == 4) add(0.f);
      else if (a.residual_type == static_cast<int>(DType::F16)) add(f16());
      else add(bf16());
    };

    f32x4 b[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) b[j] = *reinterpret_cast<const f32x4*>(bias + 16 * j);
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
      float v[4][4];
      u32x4 raw[4];
      if constexpr (kResidual) fetch_residual(step, raw);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (kGlu) {
            const int i = 2 * step + (t >> 1), j = 2 * (t & 1);
            const float g = acc[i][j][e] + b[j][e], u = acc[i][j + 1][e] + b[j + 1][e];
            v[t][e] = (A == Act8::Geglu ? gelu8(g) : silu8(g)) * u;
          } else {
            const float x = acc[step][t][e] + b[t][e];
            v[t][e] = A == Act8::Gelu ? gelu8(x) : A == Act8::Relu && x < 0.f ? 0.f : x;
          }
        }
      auto block_row = [&](int t) { return row_of(step, t); };
      if constexpr (kResidual) add_residual(raw, v);
      if constexpr (kF32) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int col = block_col(t) + 4 * eq;
          __builtin_amdgcn_raw_buffer_store_b128(
              __builtin_bit_cast(u32x4, f32x4{v[t][0], v[t][1], v[t][2], v[t][3]}), dst,
              col < a.cols ? block_row(t) * pitch + col * 4 : kNowhere, 0, kStream);
        }
      } else if constexpr (kE4m3) {
        // After the exchange a lane holds the 16 codes of block eq.
        const int row = block_row(0) + (kGlu ? (eq >> 1) * 16 : 0), col = col0 + (kGlu ? eq & 1 : eq) * 16;
        unsigned s[2], q[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = 0.f;
#pragma unroll
          for (int e = 0; e < 8; e += 2) top = largest(top, v[2 * h + (e >> 2)][e & 3], v[2 * h + (e >> 2)][(e & 3) + 1]);
          s[h] = scale8(group_max(magnitude(top)));
          q[2 * h] = encode8(v[2 * h][0], v[2 * h][1], v[2 * h][2], v[2 * h][3], s[h]);
          q[2 * h + 1] = encode8(v[2 * h + 1][0], v[2 * h + 1][1], v[2 * h + 1][2], v[2 * h + 1][3], s[h]);
        }
        transpose4(q);
        const bool in = col < span;
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{q[0], q[1], q[2], q[3]}, dst, in ? row * pitch + col : kNowhere, 0, kStream);
        __builtin_amdgcn_raw_buffer_store_b8(static_cast<unsigned char>(eq & 2 ? s[1] : s[0]), dst_scales,
                                             in && !(eq & 1) ? row * (span / kBlock8) + col / kBlock8 : kNowhere, 0, 0);
      } else {
        // Two neighbouring blocks a store: after the exchange a lane holds 8 consecutive columns of the 32, and a row's
        // four lanes 64 bytes.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          unsigned x[2] = {pack16(a.out_type, v[2 * h][0], v[2 * h][1]), pack16(a.out_type, v[2 * h][2], v[2 * h][3])};
          unsigned y[2] = {pack16(a.out_type, v[2 * h + 1][0], v[2 * h + 1][1]), pack16(a.out_type, v[2 * h + 1][2], v[2 * h + 1][3])};
          pair_chunks(x[0], y[0]);
          pair_chunks(x[1], y[1]);
          const int row = block_row(2 * h), col = block_col(2 * h) + eq * 8;
          __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], x[1], y[0], y[1]}, dst, col < a.cols ? row * pitch + col * 2 : kNowhere, 0,
                                                 kStream);
        }
      }
    }
    if (!has_next) break;
    id = nid;
    nid += G;
    cur = nxt;
    has_next = nid < total;
    if (has_next) nxt = open(nid);
    half ^= 1;
    issue_bias(half);
    read_first();
  }
  // The last slabs' clamped loads may still be landing in this workgroup's LDS.
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
}

constexpr int kTileLds8[] = {
#define LAYA_T(ID, BM, BN, WM, WN, KG, SL, S, FAST, OCC, L, B, C) lds8<BM, BN, KG, SL, S>(),
    LAYA_LINEAR8_TILES
#undef LAYA_T
};

typedef void (*RingKernel)(Linear8Args, RingWalk);
RingKernel ring_kernel(Act8 act, Out8 out, bool exact, bool residual) {
  auto with = [exact, residual](auto act_c, auto out_c) -> RingKernel {
    constexpr Act8 A = decltype(act_c)::value;
    constexpr Out8 O = decltype(out_c)::value;
    if constexpr (O != Out8::F32)
      if (!exact) return residual ? linear8_ring_kernel<A, O, false, true> : linear8_ring_kernel<A, O, false, false>;
    return residual ? linear8_ring_kernel<A, O, true, true> : linear8_ring_kernel<A, O, true, false>;
  };
  auto of = [&](auto act_c) -> RingKernel {
    return out == Out8::Half   ? with(act_c, std::integral_constant<Out8, Out8::Half>())
           : out == Out8::E4m3 ? with(act_c, std::integral_constant<Out8, Out8::E4m3>())
                               : with(act_c, std::integral_constant<Out8, Out8::F32>());
  };
  switch (act) {
#define LAYA_A(A) case Act8::A: return of(std::integral_constant<Act8, Act8::A>());
    LAYA_A(Gelu) LAYA_A(Relu) LAYA_A(Geglu) LAYA_A(Swiglu)
    default: LAYA_A(None)
#undef LAYA_A
  }
}
Out8 out_of(const Linear8Args& a) {
  return a.out_type == kE4M3 ? Out8::E4m3 : a.out_type == static_cast<int>(DType::F32) ? Out8::F32 : Out8::Half;
}
RingWalk walk_of(const Linear8Args& a) {
  const long long span = a.out_type == kE4M3 ? padded8(a.cols) : a.cols, oc = gated(a.act) ? 128 : 256;
  return ring_walk((span + oc - 1) / oc, (static_cast<long long>(a.M) + 255) / 256);
}
Problem8 problem_of(const Linear8Args& a, bool exact) {
  const bool out8 = a.out_type == kE4M3;
  return Problem8{a.M, out8 ? padded8(a.cols) : a.cols, a.ld / 128, gated(a.act), out8,
                  exact || a.out_type == static_cast<int>(DType::F32), a.wide && walk_of(a).total > 0};
}

}  // namespace

bool linear8_tile_valid(int id, const Linear8Args& a) { return tile8_valid(id, problem_of(a, false)); }

int linear8_plan(const Linear8Args& a, bool exact, int cus) { return linear8_plan(problem_of(a, exact), cus); }

hipError_t linear8_prepare() {
  hipError_t e = hipSuccess;
#define LAYA_T(ID, BM, BN, WM, WN, KG, SL, S, FAST, OCC, L, B, C)                                            \
  if (e == hipSuccess)                                                                                       \
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&linear8_kernel<BM, BN, WM, WN, KG, SL, S, FAST>), \
                            hipFuncAttributeMaxDynamicSharedMemorySize, kTileLds8[ID]);
  LAYA_LINEAR8_TILES
#undef LAYA_T
  for (int act = 0; act < 5; ++act)
    for (Out8 out : {Out8::Half, Out8::E4m3, Out8::F32})
      for (bool exact : {false, true})
        for (bool residual : {false, true})
          if (e == hipSuccess && (exact || out != Out8::F32))
            e = hipFuncSetAttribute(reinterpret_cast<const void*>(ring_kernel(static_cast<Act8>(act), out, exact, residual)),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, kRing8Lds);
  if (e == hipSuccess && gemm_device_cus() <= 0) e = hipErrorInvalidDevice;  // read by plans and launches, kept from here on
  return e;
}

hipError_t launch_linear8(const Linear8Args& a, int tile, hipStream_t stream) {
  if (a.M <= 0) return hipSuccess;
  if (tile == kFastRing8 || tile == kRing8) {
    const RingWalk walk = walk_of(a);
    LAYA_LAUNCH(ring_kernel(a.act, out_of(a), tile == kRing8, a.residual != nullptr), dim3(std::min(walk.total, gemm_device_cus())), dim3(512), kRing8Lds, stream, a, walk);
    return hipGetLastError();
  }
  const long long span = problem_of(a, false).span;
  auto grid = [&](int bm, int bn) {
    const long long oc = gated(a.act) ? bn / 2 : bn;
    return dim3(static_cast<unsigned>((span + oc - 1) / oc * ((static_cast<long long>(a.M) + bm - 1) / bm)));
  };
  switch (tile) {
#define LAYA_T(ID, BM, BN, WM, WN, KG, SL, S, FAST, OCC, L, B, C)                                            \
  case ID:                                                                                                   \
    LAYA_LAUNCH((linear8_kernel<BM, BN, WM, WN, KG, SL, S, FAST>), grid(BM, BN), dim3(64 * WM * WN * KG),    \
                kTileLds8[ID], stream, a);                                                                   \
    break;
    LAYA_LINEAR8_TILES
#undef LAYA_T
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace laya
