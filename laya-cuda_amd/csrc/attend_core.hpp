// Device parts that the kernels of attend.hip share: a sequence's ranges, what a row sees, a block's scores, weights and sums.
//
// A wave holds 32 query rows as the columns of S^T = K Q^T (v_mfma_f32_32x32x16, keys as rows): lane (row l % 32, g = l / 32)
// gets the scores of keys 8 (r / 4) + 4 g + r % 4 of each 32, so a row's softmax crosses lanes once (l and l ^ 32), and its 16-bit
// weights are already the B operand of O^T = V^T P^T.  V's rows lie in LDS as they lie in memory, a key each; its transpose
// comes from ds_read_b64_tr_b16, in which 16 lanes read four keys' 16 dims and each gets one dim's four keys.  Key slots e of a
// group of 16 keys are 4 g + e and 8 + 4 g + e - 4: those whose weights the lane holds.
//
// Scores live in log2 units.  A row's reference starts at kNothing and moves to a block's largest score only when the lane's
// weights pass 2^13 in sum (each is at most that, so fp16 holds it): most blocks need no maximum.  Weights are rounded to 16 bits
// for the matrix unit, and the normaliser sums the rounded ones.  Rows of references beyond 2^22 (biases of -1e9 as masks, where nothing else is
// seen yet) take another way to their weights, so that they cost the same: 16 x 1,024 tokens of 16 heads of 64 under a table that hides what lies behind each
// query by -1e9 108 us, by -1e4 118.
#pragma once

#include "attend.hpp"

#include <type_traits>

namespace laya {

constexpr float kNothing = -1.4426950e30f;  // of a row that has seen no key, its reference: a score of -1e30; scores not above it count as hidden
constexpr float kMostWeight = 8192.f;
constexpr float kLargest = 4194304.f;  // references up to here are rounded by at most 1/4, which all of a row's weights share
// Of a slope, in log2 units a key, that a step's shift may stand for: a score then loses 2^-24 of 31 keys' bias, 1e-4.  From 1e7 on a query's own key in such
// a step came out with a weight of 0.
constexpr float kSteepest = 64.f;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float pair_sum(f16x2 p, float acc) {
  return __builtin_amdgcn_fdot2(p, f16x2{1.0f16, 1.0f16}, acc, false);
}
__device__ __forceinline__ float pair_sum(bf16x2 p, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(p, bf16x2{static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)}, acc, false);
}
// A value joined with lane l ^ 32's, without LDS.
__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Over 32 rows; both halves of the wave hold the same ones.  Row rotations of 16 lanes, then two lanes by hand.
template <int kBy>
__device__ __forceinline__ int rotated16(int v) {
  return __builtin_amdgcn_update_dpp(v, v, 0x120 + kBy, 0xf, 0xf, false);  // row_ror
}
__device__ __forceinline__ int rows_min(int v) {
  v = min(v, rotated16<8>(v));
  v = min(v, rotated16<4>(v));
  v = min(v, rotated16<2>(v));
  v = min(v, rotated16<1>(v));
  return min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}
__device__ __forceinline__ int rows_max(int v) { return ~rows_min(~v); }

// LDS rows of a staged block: kPitch elements, in 16-byte chunks whose index is XORed with a function of the row.  K is read 16
// rows at one chunk (their 256-byte windows must hold 16 different positions), V four rows at four neighbouring chunks.
template <int D>
struct Block {
  static constexpr int kPitch = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  static constexpr int kChunks = kPitch / 8;
  __device__ static __forceinline__ int k_swizzle(int row) { return kPitch == 64 ? (row >> 1) & 7 : row & 15; }
  __device__ static __forceinline__ int v_swizzle(int row) { return kPitch == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
};

// A sequence's rows, cut to what the arrays hold.
struct Sequence {
  int q0, nq, k0, nk, prefix;
};
__device__ __forceinline__ Sequence sequence(const AttendArgs& a, int s) {
  Sequence r;
  r.q0 = __builtin_amdgcn_readfirstlane(a.q_starts[s]);
  r.k0 = __builtin_amdgcn_readfirstlane(a.k_starts[s]);
  const int nq = __builtin_amdgcn_readfirstlane(a.q_lengths[s]), nk = __builtin_amdgcn_readfirstlane(a.k_lengths[s]);
  r.nq = r.q0 < 0 || r.q0 >= a.q_rows ? 0 : max(0, min(min(nq, a.max_q), a.q_rows - r.q0));
  r.nk = r.k0 < 0 || r.k0 >= a.k_rows ? 0 : max(0, min(min(nk, a.max_k), a.k_rows - r.k0));
  r.prefix = a.prefix ? max(0, min(__builtin_amdgcn_readfirstlane(a.prefix[s]), r.nk)) : 0;
  return r;
}

// The keys that query i of a sequence sees: those below `prefix`, and [lo, hi).
struct Seen {
  int position, lo, hi;
};
__device__ __forceinline__ Seen seen(const AttendArgs& a, const Sequence& s, int i) {
  Seen r;
  r.position = i + s.nk - s.nq;
  r.lo = a.before >= 0 ? max(0, r.position - a.before) : 0;
  r.hi = a.after >= 0 ? min(s.nk, r.position + a.after + 1) : s.nk;
  if (a.bounds) {
    const int2 b = a.bounds[s.q0 + i];
    r.lo = max(r.lo, b.x);
    r.hi = min(r.hi, b.y);
  }
  if (r.lo >= r.hi) r.lo = r.hi = 0;
  if (r.lo <= s.prefix) {  // one range
    r.lo = 0;
    r.hi = max(r.hi, s.prefix);
  }
  return r;
}

// What a wave's rows see together: keys behind the prefix that some row sees lie in [lo, hi), keys that every row sees hold
// [all_lo, all_hi).  Queries first .. last; without bounds both ends grow with the query, so its two ends say it.
struct Range {
  int lo, hi, all_lo, all_hi;
};
__device__ __forceinline__ Range wave_range(const AttendArgs& a, const Sequence& s, const Seen& mine, bool valid, int first, int last) {
  Range r;
  if (a.bounds) {
    const bool any = valid && mine.lo < mine.hi;
    r.lo = rows_min(any ? mine.lo : INT_MAX);
    r.hi = rows_max(any ? mine.hi : 0);
    r.all_lo = rows_max(valid ? mine.lo : 0);
    r.all_hi = rows_min(valid ? mine.hi : INT_MAX);
  } else {
    const int p = first + s.nk - s.nq, e = last + s.nk - s.nq;
    r.lo = a.before >= 0 ? max(0, p - a.before) : 0;
    r.hi = a.after >= 0 ? max(0, min(s.nk, e + a.after + 1)) : s.nk;
    r.all_lo = a.before >= 0 ? max(0, e - a.before) : 0;
    r.all_hi = a.after >= 0 ? min(s.nk, p + a.after + 1) : s.nk;
  }
  return r;
}

// The blocks of KB keys that hold a seen key: those of the prefix, then those of a range behind it; and the order in which
// they are taken, from the one that holds key `start` down, then up from it.
template <int KB>
struct Blocks {
  int first, second, count;  // blocks of the prefix; the range's first block; all
  int turn;                  // blocks up to the starting one, less 1
  __device__ __forceinline__ Blocks(int prefix, int lo, int hi, int start) {
    first = (prefix + KB - 1) / KB;
    second = max(first, lo / KB);
    count = first + (lo < hi ? max(0, (hi + KB - 1) / KB - second) : 0);
    const int b = max(start, 0) / KB;
    turn = min(b < first ? b : max(first - 1, b - second + first), count - 1);
  }
  __device__ __forceinline__ int key(int j) const { return (j < first ? j : second + j - first) * KB; }
  __device__ __forceinline__ int taken(int t) const { return key(t <= turn ? turn - t : t); }
};

// A head's rows as the blocks' loads take them.  What lies behind a block's last row reads as zeros.
template <int KB>
struct Source {
  uint64_t base;
  unsigned row;         // bytes
  unsigned full, last;  // bytes of a whole block and of the sequence's last one
  template <typename T>
  __device__ __forceinline__ Source(const T* head, long long stride, int nk, int dim) {
    base = reinterpret_cast<uint64_t>(head);
    row = 2u * static_cast<unsigned>(stride);
    full = (KB - 1) * row + 2u * dim;
    last = (nk - 1) % KB * row + 2u * dim;
  }
  __device__ __forceinline__ i32x4 resource(int key, int nk) const {
    const uint64_t p = base + static_cast<uint64_t>(static_cast<unsigned>(key)) * row;
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(p));
    r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>(p >> 32) & 0xffff);
    r[2] = __builtin_amdgcn_readfirstlane(key + KB <= nk ? full : last);
    r[3] = 0x00020000;
    asm volatile("s_nop 4" : "+s"(r));  // a load may read an SGPR that a vector instruction wrote only five wait states later
    return r;
  }
};
constexpr unsigned kNoChunk = 0x80000000u;  // an offset behind every resource (they span fewer than 2^31 bytes)

typedef __attribute__((address_space(3))) const char* LdsBytes;
typedef __attribute__((address_space(3))) const float* LdsFloats;

// Per-lane state of 32 rows.
template <typename T, int D, int KB, bool kCap, DistanceBias kBias>
struct Rows {
  typedef typename Vec8<T>::type T8;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  typedef Block<D> B;
  static constexpr int KS = D / 16, DT = D / 32, KT = KB / 32;

  T8 q[KS];
  f32x16 o[DT];
  float reference, total;
  float top;   // what the reference was rounded from: in units of t, capped ones centred
  bool large;  // of the wave: some row's reference is larger than kLargest
  int lo, hi, prefix, position;
  float slope;  // in units of t
  int lane, g;
  unsigned k_at, v_at;  // byte offsets of this lane's first fragments

  __device__ __forceinline__ void start(int l) {
    lane = l;
    g = l >> 5;
    const int ql = l & 31;
    k_at = 2u * static_cast<unsigned>(ql * B::kPitch + ((g ^ B::k_swizzle(ql)) << 3));
    const int row = 4 * g + ((l & 15) >> 2), chunk = 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
    v_at = 2u * static_cast<unsigned>(row * B::kPitch + ((chunk ^ B::v_swizzle(row)) << 3) + (l & 1) * 4);
    reference = kNothing;
    total = 0.f;
    top = 0.f;
    large = false;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  }

  // Q^T fragments: dims 16 ks + 8 g .. + 7 of the row; zeros behind the head's last and in rows that are none.
  __device__ __forceinline__ void load_q(const T* row, int dim, bool valid) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int at = 16 * ks + 8 * g;
      if (valid && at < dim) {
        q[ks] = *reinterpret_cast<const T8*>(row + at);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[ks][e] = to_half<T>(0.f);
      }
    }
  }

  // offset: of the block behind `k` (and of its values behind `v`), a multiple of 1 KB.
  __device__ __forceinline__ void scores(LdsBytes k, unsigned offset, f32x16 (&s)[KT]) const {
    typedef __attribute__((address_space(3))) const T8* Lds8;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kt][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[kt] = mfma32(*(Lds8)(k + ((k_at + offset) ^ (ks * 32u)) + kt * 64 * B::kPitch), q[ks], s[kt]);
    }
  }

  __device__ __forceinline__ void weigh(LdsBytes v, unsigned offset, const T8 (&p)[2 * KT]) {  // O^T += V^T P^T
    typedef __attribute__((address_space(3))) s16x4* Lds4;
#pragma unroll
    for (int c = 0; c < 2 * KT; ++c)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const LdsBytes at = v + ((v_at + offset) ^ (d * 64u)) + c * 32 * B::kPitch;
        const s16x4 first = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(at));
        const s16x4 second = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(at + 16 * B::kPitch));
        const s16x8 both = __builtin_shufflevector(first, second, 0, 1, 2, 3, 4, 5, 6, 7);
        o[d] = mfma32(__builtin_bit_cast(T8, both), p[c], o[d]);
      }
  }

  // Key of score r of tile kt of the block at `key`, less the lane's first.
  static constexpr int slot(int kt, int r) { return 32 * kt + 8 * (r >> 2) + (r & 3); }

  // A block's scores stand as t, of which the log2 score is a.unit (t + shift.bias) + shift.rest: raw products, or, capped, the
  // reciprocals in cap tanh(x) = cap - 2 cap / (1 + exp(2 x)), exact to 2^-20 of the cap; biases are added in units of t.  A weight's exponent
  // is then one multiplication and addition away.  Slopes of a block to one side of every row are linear in the key: what they have in
  // common goes into the shift.  Equal scores must come out equal however large their bias is, whether it was added to t or stands in the shift: the product
  // with a.unit is not rounded by itself, and under a table capped scores are centred before their bias comes.
  // table: of this row's head, at distance 0; one in LDS is in units of t and may be read up to a block and 32 rows past the span.
  // side: -1 and 1 where all keys lie before or behind all rows' positions (or at them), 0 where not.
  struct Shift {
    float bias, rest;
  };
  template <typename Table>
  __device__ __forceinline__ Shift change(const AttendArgs& a, f32x16 (&s)[KT], int key, Table table, int side) const {
    capped(a, s);
    Shift shift{0.f, kCap ? a.cap : 0.f};
    const int at = key + 4 * g - position;
    if constexpr (kBias == DistanceBias::Slopes) {
      const float from = static_cast<float>(at);
      if (side) {
        const float by = side < 0 ? -slope : slope;  // of |d| = -d or d
        shift.bias = from * by;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kt][r] += static_cast<float>(slot(kt, r)) * by;
      } else {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kt][r] = __builtin_fmaf(fabsf(from + static_cast<float>(slot(kt, r))), slope, s[kt][r]);
      }
    }
    if constexpr (kBias == DistanceBias::Table) {
      shift.rest = 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = at + slot(kt, r);
          const float t = kCap ? s[kt][r] - 0.5f : s[kt][r];
          if constexpr (std::is_same<Table, LdsFloats>::value) s[kt][r] = t + table[d];
          else s[kt][r] = __builtin_fmaf(table[max(-a.span, min(a.span, d))], a.per_unit, t);
        }
    }
    return shift;
  }
  __device__ __forceinline__ void capped(const AttendArgs& a, f32x16 (&s)[KT]) const {
    if constexpr (kCap) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kt][r] = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[kt][r] * a.scale) + 1.0f);
    }
  }

  // Scores of hidden keys: none.  A lane's keys of a step are bits of one word, and a score takes two instructions.
  __device__ __forceinline__ void hide(f32x16 (&s)[KT], int key) const {
    static_assert(KT == 1, "32 keys a step");
    const auto below = [&](int end) {  // keys before `end`
      const int n = end - key;
      return n <= 0 ? 0u : ~0u >> (32 - min(n, 32));
    };
    const unsigned hidden = ~((below(hi) & ~below(lo)) | below(prefix)) >> (4 * g);
    constexpr int kNone = kCap ? 0x7f800000 : static_cast<int>(0xff800000);  // infinite, towards a score of -infinity
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int mask = __builtin_amdgcn_sbfe(static_cast<int>(hidden), slot(0, r), 1);
      s[0][r] = __int_as_float((mask & kNone) | (~mask & __float_as_int(s[0][r])));
    }
  }

  // The largest score, in units of t, capped ones centred: of the largest t, or of the smallest where the cap's unit is negative.
  __device__ __forceinline__ float block_top(const f32x16 (&s)[KT], Shift shift) const {
    float m = kCap ? INFINITY : -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = kCap ? fminf(m, s[kt][r]) : fmaxf(m, s[kt][r]);
    m = m - centre(shift) + shift.bias;
    return kCap ? -halves_max(-m) : halves_max(m);
  }
  __device__ __forceinline__ static float centre(Shift shift) { return kCap && shift.rest != 0.f ? 0.5f : 0.f; }
  __device__ __forceinline__ bool is_large() const { return fabsf(reference) > kLargest && reference > kNothing; }

  // kLarge: rows of large references subtract what those were rounded from, in units of t, which equal scores have in common to the last bit; a
  // rounded one is off by whole powers of two from 2^24 on, which would take every weight to 0 or past the type.
  template <bool kLarge>
  __device__ __forceinline__ float weights(const AttendArgs& a, const f32x16 (&s)[KT], T8 (&p)[2 * KT], Shift shift) const {
    float sum[2] = {0.f, 0.f};
    float base = __builtin_fmaf(shift.bias, a.unit, -reference), from = 0.f;
    if constexpr (kCap) base += shift.rest;
    if (kLarge && is_large()) {
      base = 0.f;
      from = top - shift.bias + centre(shift);
    }
#pragma unroll
    for (int c = 0; c < 2 * KT; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float t = s[c >> 1][8 * (c & 1) + e];
        p[c][e] = to_half<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(kLarge ? t - from : t, a.unit, base)));
      }
      sum[0] = pair_sum(__builtin_shufflevector(p[c], p[c], 0, 1), sum[0]);
      sum[1] = pair_sum(__builtin_shufflevector(p[c], p[c], 2, 3), sum[1]);
      sum[0] = pair_sum(__builtin_shufflevector(p[c], p[c], 4, 5), sum[0]);
      sum[1] = pair_sum(__builtin_shufflevector(p[c], p[c], 6, 7), sum[1]);
    }
    return sum[0] + sum[1];
  }

  // The first block of a wave: its largest score is the reference, before any weight is made.
  __device__ __forceinline__ void open(const AttendArgs& a, const f32x16 (&s)[KT], Shift shift) {
    top = block_top(s, shift);
    reference = fmaxf(kNothing, top * a.unit);
    large = __builtin_amdgcn_ballot_w64(is_large()) != 0;
  }

  // A step's weights and their sum.  Where they are too large for the reference, it moves to the step's largest score.
  __device__ __forceinline__ float weigh_step(const AttendArgs& a, const f32x16 (&s)[KT], T8 (&p)[2 * KT], Shift shift) {
    float sum = INFINITY;
    if (!large) sum = weights<false>(a, s, p, shift);
    if (__builtin_amdgcn_ballot_w64(!(sum <= kMostWeight))) {
      const float t = block_top(s, shift), m = t * a.unit;
      const bool was_large = is_large();
      const bool moves = was_large && fabsf(m) > kLargest ? (kCap ? t < top : t > top) : m > reference + 8.f;
      const float by = was_large ? (top - t) * a.unit : reference - m;
      const float alpha = moves ? __builtin_amdgcn_exp2f(by) : 1.f;
      if (moves) {
        reference = m;
        top = t;
      }
      large = __builtin_amdgcn_ballot_w64(is_large()) != 0;
      total *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      sum = weights<true>(a, s, p, shift);
    }
    return sum;
  }

  // Rows (bits 0 to 31) to be done again by themselves: those whose sums are no numbers (a weight of 0 times an infinity or NaN in a
  // hidden key's value, if nothing the row sees is one), and those whose weights are all too small, where biases of more than 2^24 in several steps' shifts
  // were rounded apart.
  __device__ __forceinline__ unsigned doubtful(float row_total) const {
    float sum[4] = {total, 0.f, 0.f, 0.f};  // NaN for a NaN or an infinity
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[r & 3] = __builtin_fmaf(o[d][r], 0.f, sum[r & 3]);
    const float x = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    const unsigned long long bad = __builtin_amdgcn_ballot_w64(x != x || (row_total < 0.5f && reference > kNothing));
    return static_cast<unsigned>(bad | bad >> 32);
  }
};

// One row by itself, hidden keys never touched and the reference taken from each rounded score: what a wave does for a doubtful row.  Blocks [j0, j1) of
// the row's tile; lane l holds dims l, l + 64, ...
template <typename T, int D, int KB, bool kCap, DistanceBias kBias>
struct CarefulRow {
  static constexpr int ND = (D + 63) / 64;
  float sum[ND], reference, total;

  __device__ __forceinline__ void run(const AttendArgs& a, const T* q, const T* k, const T* v, int nk, int position, int lo, int hi,
                                      int prefix, float slope, const float* table, const Blocks<KB>& blocks, int j0, int j1, int lane) {
    typedef typename Vec8<T>::type T8;
    reference = kNothing;
    total = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) sum[i] = 0.f;
    for (int j = j0; j < j1; ++j) {
      const int first = blocks.taken(j), key = first + lane;
      const bool see = lane < KB && key < nk && ((key >= lo && key < hi) || key < prefix);
      float x = -INFINITY;
      if (see) {
        const T* row = k + key * a.k_row;
        x = 0.f;
        for (int c = 0; c < a.dim; c += 8) {
          const T8 kc = *reinterpret_cast<const T8*>(row + c), qc = *reinterpret_cast<const T8*>(q + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) x = __builtin_fmaf(to_float(kc[e]), to_float(qc[e]), x);
        }
        if constexpr (kCap) x = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * a.scale) + 1.0f) - 0.5f;
        // A slope past the type's range in units of a raw score is infinite here, and 0 times it no number, which is what brings the row here.
        if constexpr (kBias == DistanceBias::Slopes) x = key == position ? x : __builtin_fmaf(fabsf(static_cast<float>(key - position)), slope, x);
        if constexpr (kBias == DistanceBias::Table) x = __builtin_fmaf(table[max(-a.span, min(a.span, key - position))], a.per_unit, x);
        x *= a.unit;
      }
      const float to = fmaxf(reference, wave_max(x));
      const float alpha = to == reference ? 1.f : __builtin_amdgcn_exp2f(reference - to);
      const float p = see ? __builtin_amdgcn_exp2f(x - to) : 0.f;
      reference = to;
      total = total * alpha + wave_sum(p);
#pragma unroll
      for (int i = 0; i < ND; ++i) sum[i] *= alpha;
      unsigned long long left = __builtin_amdgcn_ballot_w64(see);
      while (left) {
        const int t = __builtin_ctzll(left);
        left &= left - 1;
        const float w = __shfl(p, t, kWave);
#pragma unroll
        for (int i = 0; i < ND; ++i)
          if (lane + 64 * i < a.dim) sum[i] = __builtin_fmaf(w, to_float(v[(first + t) * a.v_row + lane + 64 * i]), sum[i]);
      }
      if (total != total) break;  // NaN from a seen score: so is every output
    }
    if (total != total) {
#pragma unroll
      for (int i = 0; i < ND; ++i) sum[i] = total;
    }
  }
};

}  // namespace laya
