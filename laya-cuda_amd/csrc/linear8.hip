// Matrix product of 8-bit rows: out = act(x w^T + bias) + residual, x [M][K] and w [N][K] in the form of rows8.hpp.
//
// linear8_kernel keeps every product exact: a code times its scale is a bf16 value (4 significant bits), so the codes
// are widened in registers, with their scales, by v_cvt_scalef32_pk_bf16_fp8 and multiplied by v_mfma_f32_16x16x32_bf16,
// whose sums are fp32 (measured: 8e-8 of the result's norm at K = 4,096).  It moves half the bytes of the 16-bit
// product, which is what few rows are bound by.
//
// Layout: whole 128-code slabs go straight from global memory into LDS, 16-byte chunk c of row r at position
// c ^ (r / 2) % 8, so that 16 lanes reading one chunk of 16 consecutive rows touch all banks once.  A workgroup
// owns BM x BN outputs, WM x WN waves of it times KG groups that split the slabs; S stages of SL slabs are in
// flight.  The groups' fp32 tiles are added in group order through LDS, so results do not depend on timing.
#include "kernels.hpp"
#include "rows8.hpp"
#include "tiles.hpp"

#include <algorithm>
#include <type_traits>

namespace laya {

namespace {

// lds_load16_buffer's form for 4 bytes a lane: lane l's dword goes to LDS byte address lds + 4 l.
__device__ __forceinline__ void lds_load4_buffer(i32x4 rsrc, unsigned voffset, unsigned soffset, unsigned lds) {
  soffset = __builtin_amdgcn_readfirstlane(soffset);
  asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(lds));
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

// Activations.  NaNs stay NaNs and +infinity stays itself.  kFine: for fp32 outputs (libm); else accurate to
// 3e-7 absolute, far inside a 16-bit rounding (see gelu16, whose argument is capped where its q has reached 0).
template <bool kFine>
__device__ __forceinline__ float gelu8(float x) {
  if constexpr (kFine) return 0.5f * x * (1.0f + erff(x * 0.7071067811865475f));
  const float t = fminf(fabsf(x), 16.f);
  return x != x ? x : gelu16(-t) + (x > 0.f ? x : 0.f);
}
template <bool kFine>
__device__ __forceinline__ float silu8(float x) {
  if constexpr (kFine) return x / (1.0f + expf(-x));
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

__host__ __device__ __forceinline__ bool gated(Act8 act) { return act == Act8::Geglu || act == Act8::Swiglu; }

// Output columns n .. n + 3 of row `row` after bias and activation: adds the residual, rounds once and stores.
// 8-bit outputs are made by 8 lanes with consecutive quads of the same row (a whole block), all of them
// calling; columns past `cols` come in as zeros and only an 8-bit row's padding is stored from them.
__device__ __forceinline__ void finish4(const Linear8Args& a, long long row, int n, float (&v)[4]) {
  const size_t at = static_cast<size_t>(row) * a.cols + n;
  const bool whole = a.vec && n < a.cols;
  if (a.residual) {
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    auto take = [&](auto zero) {
      typedef decltype(zero) T;
      typedef T T4 __attribute__((ext_vector_type(4)));
      const T* src = static_cast<const T*>(a.residual) + at;
      if (whole) {
        const T4 t = *reinterpret_cast<const T4*>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = static_cast<float>(t[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < a.cols) r[i] = static_cast<float>(src[i]);
      }
    };
    if (a.residual_type == static_cast<int>(DType::F32)) take(0.f);
    else if (a.residual_type == static_cast<int>(DType::F16)) take(f16());
    else take(bf16());
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] + r[i];
  }
  if (a.out_type == kE4M3) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned m = magnitude(v[i]);
      top = top > m ? top : m;
    }
    const unsigned s = scale8(block_top8(top));
    const size_t ld = static_cast<size_t>(padded8(a.cols));
    *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(a.out) + row * ld + n) = encode8(v[0], v[1], v[2], v[3], s);
    if (n % kBlock8 == 0) a.out_scales[row * (ld / kBlock8) + n / kBlock8] = static_cast<uint8_t>(s);
    return;
  }
  auto put = [&](auto zero) {
    typedef decltype(zero) T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T* dst = static_cast<T*>(a.out) + at;
    if (whole) {
      *reinterpret_cast<T4*>(dst) = T4{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.cols) dst[i] = static_cast<T>(v[i]);
    }
  };
  if (a.out_type == static_cast<int>(DType::F32)) put(0.f);
  else if (a.out_type == static_cast<int>(DType::F16)) put(f16());
  else put(bf16());
}

// Dwords of a slab's scales in LDS: x's rows, then w's, each in whole 64-row loads.
constexpr int scale_rows8(int rows) { return (rows + 63) / 64 * 64; }
template <int BM, int BN, int SL> constexpr int stage_bytes8() {
  return SL * ((BM + BN) * 128 + (scale_rows8(BM) + scale_rows8(BN)) * 4);
}
template <int BM, int BN, int KG, int SL, int S> constexpr int lds8() {
  const int stages = S * stage_bytes8<BM, BN, SL>(), parts = KG * BM * (BN + 4) * 4;
  return stages > parts ? stages : parts;
}

template <int BM, int BN, int WM, int WN, int KG, int SL, int S>
__global__ __launch_bounds__(64 * WM * WN * KG) void linear8_kernel(Linear8Args a) {
  constexpr int NW = WM * WN * KG, NT = 64 * NW;
  constexpr int WTM = BM / WM, WTN = BN / WN, MB = WTM / 16, NB = WTN / 16;
  static_assert(MB >= 1 && NB >= 1 && WTM % 16 == 0 && WTN % 16 == 0, "16x16 MFMA blocks");
  constexpr int PITCH = BN + 4;  // floats per row of a partial tile: 16-byte rows, spread over the banks
  constexpr int RG = (BM + BN) / 8, SX = scale_rows8(BM), SG = (SX + scale_rows8(BN)) / 64;
  constexpr int STAGE = stage_bytes8<BM, BN, SL>(), CODES = SL * (BM + BN) * 128;
  constexpr int GROUPS = SL * (RG + SG);
  constexpr int NLD = (GROUPS + NW - 1) / NW;  // loads per wave and stage; past the last, the last again
  static_assert((S - 1) * NLD < 64, "vmcnt range");
  extern __shared__ __align__(16) unsigned char smem_raw[];
  float* const red = reinterpret_cast<float*>(smem_raw);  // [KG][BM][PITCH], after the main loop

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
        const bool isx = rg * 8 < BM;
        const unsigned row = static_cast<unsigned>(isx ? r : r - BM);
        lds_load16_buffer(isx ? rsX : rsW, row * static_cast<unsigned>(a.ld) + (((lane & 7) ^ ((r >> 1) & 7)) << 4), k,
                          base + static_cast<unsigned>(g * 1024));
      } else {
        const int sg = (g - SL * RG) % SG, r = sg * 64 + lane;
        const unsigned k = static_cast<unsigned>(min(stage * SL + (g - SL * RG) / SG, n - 1)) * 4u;
        const bool isx = sg * 64 < SX;
        const unsigned row = static_cast<unsigned>(isx ? r : r - SX);
        lds_load4_buffer(isx ? rsXs : rsWs, row * static_cast<unsigned>(sld), k,
                         base + static_cast<unsigned>(CODES + (g - SL * RG) * 256));
      }
    }
  };

  const int kg = wave / (WM * WN), wm0 = (wave % (WM * WN)) / WN * WTM, wn0 = wave % WN * WTN;
  const int r16 = lane & 15, kq = lane >> 4;
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A slab's products in two halves of 64 codes: lane group kq takes the 16 codes at 16 kq of the half, which lie
  // in its block kq / 2, as two MFMA operands of 8 (any order of k will do that x and w share).
  auto compute = [&](int buf, int count) {
    constexpr int PS = (SL + KG - 1) / KG;
#pragma unroll
    for (int u = 0; u < PS; ++u) {
      const int slab = kg + u * KG;
      if (slab < count) {
        const unsigned char* const codes = smem_raw + buf * STAGE + slab * (BM + BN) * 128;
        const unsigned* const sc = reinterpret_cast<const unsigned*>(smem_raw + buf * STAGE + CODES) + slab * SG * 64;
        unsigned sx[MB], sw[NB];
#pragma unroll
        for (int i = 0; i < MB; ++i) sx[i] = sc[wm0 + i * 16 + r16] >> (8 * (kq >> 1));
#pragma unroll
        for (int j = 0; j < NB; ++j) sw[j] = sc[SX + wn0 + j * 16 + r16] >> (8 * (kq >> 1));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          auto fragment = [&](int r, unsigned s, bf16x8 (&f)[2]) {
            const i32x4 c = *reinterpret_cast<const i32x4*>(codes + r * 128 + (((4 * h + kq) ^ ((r >> 1) & 7)) << 4));
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

  float* const mine = red + kg * BM * PITCH;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      *reinterpret_cast<f32x4*>(mine + (wm0 + i * 16 + r16) * PITCH + wn0 + j * 16 + 4 * kq) = acc[i][j];
  __syncthreads();

  // Four columns n .. n + 3 of tile row r: the groups' sum in group order, and the bias; zeros past N.
  auto total4 = [&](int r, int n, float (&v)[4]) {
    f32x4 t = *reinterpret_cast<const f32x4*>(red + r * PITCH + n);
#pragma unroll
    for (int w = 1; w < KG; ++w) {
      const f32x4 o = *reinterpret_cast<const f32x4*>(red + (w * BM + r) * PITCH + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = t[e] + o[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = t[e];
      if (a.bias && n0 + n + e < a.N) v[e] = v[e] + a.bias[n0 + n + e];
    }
  };
  const bool fine = a.out_type == static_cast<int>(DType::F32);
  const int quads = oc / 4;
  for (int c = tid; c < BM * quads; c += NT) {
    const int r = c / quads, f = (c % quads) * 4;
    const long long row = m0 + r;
    const int col = static_cast<int>(n0 / BN) * oc + f;
    if (row >= a.M || col >= span) continue;  // alike in the 8 lanes of a block
    float v[4];
    if (glu) {
      float g[4];
      const int n = (f / 16) * 32 + f % 16;
      total4(r, n, g);
      total4(r, n + 16, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = a.act == Act8::Geglu ? (fine ? gelu8<true>(g[e]) : gelu8<false>(g[e]))
                                             : (fine ? silu8<true>(g[e]) : silu8<false>(g[e]));
        v[e] = y * v[e];
      }
    } else {
      total4(r, f, v);
      if (a.act == Act8::Gelu) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fine ? gelu8<true>(v[e]) : gelu8<false>(v[e]);
      } else if (a.act == Act8::Relu) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
      }
    }
    finish4(a, row, col, v);
  }
}

// Tile menu: BM, BN, WM, WN, KG, SL, S.
#define LAYA_LINEAR8_TILES        \
  LAYA_T(0, 16, 64, 1, 2, 4, 4, 2) \
  LAYA_T(1, 128, 128, 2, 4, 1, 1, 3)

struct Tile8 {
  int bm, bn, lds, threads;
};
constexpr Tile8 kTiles8[] = {
#define LAYA_T(ID, BM, BN, WM, WN, KG, SL, S) {BM, BN, lds8<BM, BN, KG, SL, S>(), 64 * WM * WN * KG},
    LAYA_LINEAR8_TILES
#undef LAYA_T
};
constexpr int kTiles8Count = sizeof(kTiles8) / sizeof(kTiles8[0]);

int columns8(const Linear8Args& a, int bn) { return gated(a.act) ? bn / 2 : bn; }

}  // namespace

int linear8_tile_count() { return kTiles8Count; }

bool linear8_tile_valid(int id, const Linear8Args& a) {
  // A block of 32 output codes, and a group of 16 gate and 16 value rows, lie inside one tile.
  return id >= 0 && id < kTiles8Count && (a.out_type != kE4M3 || columns8(a, kTiles8[id].bn) % kBlock8 == 0) &&
         (!gated(a.act) || kTiles8[id].bn % 32 == 0);
}

int linear8_plan(const Linear8Args& a, int) { return a.M <= 64 ? 0 : 1; }

hipError_t linear8_prepare() {
  hipError_t e = hipSuccess;
#define LAYA_T(ID, BM, BN, WM, WN, KG, SL, S)                                                            \
  if (e == hipSuccess)                                                                                   \
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&linear8_kernel<BM, BN, WM, WN, KG, SL, S>),   \
                            hipFuncAttributeMaxDynamicSharedMemorySize, kTiles8[ID].lds);
  LAYA_LINEAR8_TILES
#undef LAYA_T
  return e;
}

hipError_t launch_linear8(const Linear8Args& a, int tile, hipStream_t stream) {
  if (a.M <= 0) return hipSuccess;
  const Tile8& t = kTiles8[tile];
  const long long span = a.out_type == kE4M3 ? padded8(a.cols) : a.cols, oc = columns8(a, t.bn);
  const long long groups = (span + oc - 1) / oc * ((static_cast<long long>(a.M) + t.bm - 1) / t.bm);
  if (groups > 0x7fffffffLL) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(groups)), block(t.threads);
  switch (tile) {
#define LAYA_T(ID, BM, BN, WM, WN, KG, SL, S) \
  case ID: LAYA_LAUNCH((linear8_kernel<BM, BN, WM, WN, KG, SL, S>), grid, block, t.lds, stream, a); break;
    LAYA_LINEAR8_TILES
#undef LAYA_T
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace laya
