// Attention over packed sequences: prompts, single tokens and what lies between (attend_core.hpp has what they share).
//
// Compiled once for each head width (LAYA_ATTEND_DIM), and once without for what is no kernel of a width.
#include "attend_core.hpp"

#include <type_traits>

namespace laya {

#ifdef LAYA_ATTEND_DIM

namespace {

constexpr int kPad = 96;  // distances past a bias table's span that the scores of a block near its ends reach: its 64 keys and 32 rows

// Prompts: a workgroup of NW waves owns 32 NW queries of one head, and blocks of 64 keys pass through LDS, shared by the waves
// and double-buffered.  A wave works on them 32 keys at a time (scores, weights, products with V: one pass over the keys with the
// running reference and total) and skips those that none of its rows sees.
//
// What bounds it: the card's power and the vector instructions beside the matrix ones.  64 x 1,024 tokens of 16 heads of 64 run
// 350 us (785 TFLOP/s; boxes differ, 316 to 362) at 1.91 of 2.4 GHz with the matrix cores busy 41% of the cycles and vector instructions 62%; with zeros for
// inputs 280 us.  Copies without the exponentials, the loads or one of the products run 320, 315 and 290 us.  16,384
// causal tokens of 8 heads of 128: 511 to 545 us, 1.01 to 1.08 PFLOP/s, the matrix cores 46%.
// Why 32 keys a step in one straight line, with 102 to 114 registers for heads of 64: four such workgroups share a CU (up to 128).  64 keys a
// step took 373 us where this took 361, scores of the next step under the softmax of this one 388 against 352, two row groups a
// wave (half the LDS reads) 354 against 349 for heads of 64 and 1,535 against 1,069 for 128, three buffers 382 against 344, blocks of 32
// keys 394 against 350, raised priorities for either phase or by slot nothing.  Tiles of 64 queries, two waves: 488 against 338, documents 314
// against 239, ragged requests with a bias table 121 against 83, 1,571 tokens behind a window of heads of 80 64 against 41.
template <typename T, int D, bool kCap, DistanceBias kBias, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(D <= 64 || (D == 96 && NW == 8) ? 4 : 2))) void attend_kernel(
    AttendArgs a, int tiles, int unit, int units) {
  constexpr int NT = 64 * NW, TR = 32 * NW, KB = 64, P = Block<D>::kPitch, kChunks = P / 8;
  constexpr int SB = 32;  // keys of one step
  typedef Rows<T, D, SB, kCap, kBias> R;
  typedef typename R::T8 T8;
  typedef typename Vec4<T>::type T4;
  // Workgroup -> (sequence, head, tile).  Workgroups go round the 8 XCDs by their number: a unit (the tiles of one head, or of
  // the heads that share keys) stays on one XCD, so that its keys come into one L2 once; tiles with the most keys first.
  int pair, tile;
  {
    const int id = blockIdx.x;
    if (unit) {
      const int y = id >> 3, at = y / (tiles * unit), w = y - at * tiles * unit;
      const int u = (id & 7) + 8 * at;
      if (u >= units) return;
      const int t = w / unit;
      tile = tiles - 1 - t;
      pair = u * unit + (w - t * unit);
    } else {
      const int t = id / units;
      tile = tiles - 1 - t;
      pair = id - t * units;
    }
  }
  const int s = pair / a.heads;
  const int head = pair - s * a.heads, kv = head / a.group;
  const Sequence sq = sequence(a, s);
  const int row0 = tile * TR;
  if (row0 >= sq.nq) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = row0 + wave * 32 + (lane & 31);
  const bool valid = i < sq.nq;
  const bool active = row0 + wave * 32 < sq.nq;  // waves past the last query only stage keys
  const Seen me = valid ? seen(a, sq, i) : Seen{i + sq.nk - sq.nq, 0, 0};

  __shared__ __align__(16) T skv[4][KB * P];  // two buffers of K, two of V
  __shared__ Range wg_range[NW];
  extern __shared__ float stable[];  // the head's bias table in units of t, 2 (span + kPad) + 1

  const Range range = wave_range(a, sq, me, valid, row0 + wave * 32, min(row0 + wave * 32 + 31, sq.nq - 1));
  if (lane == 0) wg_range[wave] = active ? range : Range{INT_MAX, 0, 0, INT_MAX};
  if constexpr (kBias == DistanceBias::Table) {
    const float* from = a.table + static_cast<size_t>(head) * (2 * a.span + 1);
    for (int e = tid; e < 2 * (a.span + kPad) + 1; e += NT) stable[e] = from[max(0, min(2 * a.span, e - kPad))] * a.per_unit;
  }
  __syncthreads();
  Range wg = wg_range[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    wg.lo = min(wg.lo, wg_range[w].lo);
    wg.hi = max(wg.hi, wg_range[w].hi);
    wg.all_lo = max(wg.all_lo, wg_range[w].all_lo);
    wg.all_hi = min(wg.all_hi, wg_range[w].all_hi);
  }
  // With a bias the keys next to the queries come first: their scores are the largest as a rule, and references move once.
  const int last_position = min(row0 + TR - 1, sq.nq - 1) + sq.nk - sq.nq;
  const Blocks<KB> blocks(sq.prefix, __builtin_amdgcn_readfirstlane(wg.lo), __builtin_amdgcn_readfirstlane(wg.hi),
                          kBias == DistanceBias::None ? 0 : last_position);
  const int plain_lo = __builtin_amdgcn_readfirstlane(wg.all_lo), plain_hi = __builtin_amdgcn_readfirstlane(wg.all_hi) - KB;
  const int nb = blocks.count;

  const T* K = static_cast<const T*>(a.k) + sq.k0 * a.k_row + kv * a.k_head;
  const T* V = static_cast<const T*>(a.v) + sq.k0 * a.v_row + kv * a.v_head;
  const T* Q = static_cast<const T*>(a.q) + (sq.q0 + (valid ? i : 0)) * a.q_row + head * a.q_head;

  // This thread's 16-byte chunks of a block: row r0 + step m, chunk index swizzled by the row.
  constexpr int CH = KB * kChunks / NT, step = NT / kChunks;
  const int r0 = tid / kChunks, c0 = tid % kChunks;
  unsigned at_k[CH], at_v[CH];
#pragma unroll
  for (int m = 0; m < CH; ++m) {
    const int r = r0 + m * step, ck = c0 ^ Block<D>::k_swizzle(r), cv = c0 ^ Block<D>::v_swizzle(r);
    at_k[m] = ck * 8 < a.dim ? 2u * static_cast<unsigned>(r) * static_cast<unsigned>(a.k_row) + 16u * ck : kNoChunk;
    at_v[m] = cv * 8 < a.dim ? 2u * static_cast<unsigned>(r) * static_cast<unsigned>(a.v_row) + 16u * cv : kNoChunk;
  }
  const Source<KB> from_k(K, a.k_row, sq.nk, a.dim), from_v(V, a.v_row, sq.nk, a.dim);
  constexpr unsigned kBuffer = KB * P * sizeof(T);
  const unsigned lds_k = lds_address(skv[0]) + wave * 1024u, lds_v = lds_address(skv[2]) + wave * 1024u;
  auto load = [&](int key, unsigned buffer) __attribute__((always_inline)) {
    const i32x4 rk = from_k.resource(key, sq.nk), rv = from_v.resource(key, sq.nk);
#pragma unroll
    for (int m = 0; m < CH; ++m) lds_load16_buffer<true>(rk, at_k[m], 0u, lds_k + buffer + NT * 16u * m);
#pragma unroll
    for (int m = 0; m < CH; ++m) lds_load16_buffer<true>(rv, at_v[m], 0u, lds_v + buffer + NT * 16u * m);
  };

  R rows;
  rows.start(lane);
  int key0 = blocks.taken(0);
  if (nb > 0) load(key0, 0);
  rows.load_q(Q, a.dim, valid);
  rows.lo = me.lo;
  rows.hi = me.hi;
  rows.prefix = sq.prefix;
  rows.position = me.position;
  rows.slope = kBias == DistanceBias::Slopes ? -a.slopes[head] * a.per_unit : 0.f;
  const LdsFloats table = (LdsFloats)(stable) + a.span + kPad;

  float far_left = 0.f, far_right = 0.f;
  if constexpr (kBias == DistanceBias::Table) {
    far_left = stable[0];
    far_right = stable[2 * (a.span + kPad)];
  }
  const int first_position = __builtin_amdgcn_readfirstlane(me.position);
  const bool steep = kBias == DistanceBias::Slopes && !(fabsf(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(rows.slope))) * a.unit) <= kSteepest);
  unsigned buffer = 0;
  bool fresh = true;  // no step done
  for (int j = 0; j < nb; ++j, buffer ^= kBuffer) {
    publish_stage<waitcnt_vm(0)>();
    const int now = key0;
    if (j + 1 < nb) {
      key0 = blocks.taken(j + 1);
      load(key0, buffer ^ kBuffer);
    }
    if (!active) continue;
    const bool plain = now >= plain_lo && now <= plain_hi;  // every wave's rows see every key
#pragma unroll
    for (int h = 0; h < KB / SB; ++h) {
      const int key = now + SB * h;
      bool whole = true;
      if (!plain) {
        whole = key + SB <= sq.prefix || (key >= range.all_lo && key + SB <= range.all_hi);
        if (!(whole || key < sq.prefix || (key < range.hi && key + SB > range.lo))) continue;
      }
      f32x16 t[R::KT];
      T8 p[2 * R::KT];
      rows.scores((LdsBytes)(skv[0]), buffer + SB * h * P * 2u, t);
      typename R::Shift shift;
      const int first = key - first_position;  // of the wave's first query to the step's first key
      if (kBias == DistanceBias::Table && (first + SB - 1 <= -a.span || first - 31 >= a.span)) {
        // Steps wholly past the span on one side have one bias; the table's LDS rows reach as far as the others need.
        rows.capped(a, t);
        shift = {first < 0 ? far_left : far_right, kCap ? a.cap : 0.f};
      } else {
        shift = rows.change(a, t, key, table, steep ? 0 : first + SB - 1 <= 0 ? -1 : first - 31 >= 0 ? 1 : 0);
      }
      if (!whole) rows.hide(t, key);
      if (fresh) rows.open(a, t, shift);
      fresh = false;
      rows.total += rows.weigh_step(a, t, p, shift);
      rows.weigh((LdsBytes)(skv[2]), buffer + SB * h * P * 2u, p);
    }
  }
  if (!active) return;

  T* out = static_cast<T*>(a.out) + head * a.out_head;
  const unsigned live = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(valid));
  const float total = halves_sum(rows.total);
  unsigned bad = rows.doubtful(total) & live;
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  if (valid && !(bad >> (lane & 31) & 1)) {
    T* row = out + (sq.q0 + i) * a.out_row;
#pragma unroll
    for (int d = 0; d < R::DT; ++d)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int at = 32 * d + 8 * r4 + 4 * rows.g;
        T4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to_half<T>(rows.o[d][4 * r4 + e] * inv);
        if (at < a.dim) *reinterpret_cast<T4*>(row + at) = v;
      }
  }
  while (bad) {
    const int b = __builtin_ctz(bad);
    bad &= bad - 1;
    const int ib = row0 + wave * 32 + b;
    const Seen m = seen(a, sq, ib);
    CarefulRow<T, D, KB, kCap, kBias> c;
    c.run(a, static_cast<const T*>(a.q) + (sq.q0 + ib) * a.q_row + head * a.q_head, K, V, sq.nk, m.position, m.lo, m.hi, sq.prefix,
          rows.slope, a.table ? a.table + static_cast<size_t>(head) * (2 * a.span + 1) + a.span : nullptr, blocks, 0, nb, lane);
    const float n = c.total == 0.f ? 0.f : 1.0f / c.total;
#pragma unroll
    for (int x = 0; x < c.ND; ++x)
      if (lane + 64 * x < a.dim) out[(sq.q0 + ib) * a.out_row + lane + 64 * x] = to_half<T>(c.sum[x] * n);
  }
}

// Few rows: a workgroup owns 32 rows, the (token, head) pairs of the heads that share keys, and its waves split their keys into
// blocks of 32 (eight waves, four for heads above 128), each wave with a place of its own in LDS for a block of K and one of V.  The next K is on its way from the
// scores to the next ones, the next V from one product to the next.  Long contexts are shared by a.splits workgroups, whose sums
// join_kernel adds in a fixed order.
//
// What bounds it: over long caches their bytes (4 tokens over 131,072 keys of 8 heads of 128: 381 us and 4 to join, 5.6 TB/s where a copy
// reaches 4.8; 48 ragged ones over up to 4,100 keys of 16 heads of 64: 97 us, 4.6 TB/s), over short ones a launch and five dependent
// steps (kernel arguments, lengths, keys, sums in LDS, output): 500 keys 6.8 us, of which an empty kernel takes 2.2.
// Why eight waves with one place each, not four with two: as many bytes on their way, and half the rounds (30,000 keys of 8 heads
// 69 -> 29 us with as many workgroups as compute units, 500 keys 9.5 -> 8.3).
template <int D>
constexpr int split_waves() {
  return D <= 128 ? 8 : 4;  // what 128 KB of LDS hold, or for heads of 64 half of it
}
template <typename T, int D, bool kCap, DistanceBias kBias>
__global__ __launch_bounds__(64 * split_waves<D>()) __attribute__((amdgpu_waves_per_eu(D <= 64 ? 4 : D <= 128 ? 2 : 1))) void attend_split_kernel(
    AttendArgs a, int units) {
  constexpr int KB = 32, NW = split_waves<D>(), NT = 64 * NW, P = Block<D>::kPitch, kChunks = P / 8;
  typedef Rows<T, D, KB, kCap, kBias> R;
  typedef typename R::T8 T8;
  typedef typename Vec4<T>::type T4;
  constexpr int kPlace = 2 * KB * P;  // elements of a wave's place: a block of K, one of V
  constexpr int OP = D + 4;           // pitch of a row of sums (floats): 16 rows' quads lie in 16 places of 256 bytes
  constexpr size_t kPlaces = NW * kPlace * sizeof(T), kSums = NW * 32 * OP * sizeof(float);
  __shared__ __align__(16) char lds[kPlaces > kSums ? kPlaces : kSums];
  __shared__ float s_reference[NW][32], s_total[NW][32];
  __shared__ int s_bad[32];

  // Workgroup -> (sequence, key head, tile, split).  The divisions are scalar code of some 100 cycles each, before anything can be
  // loaded.  Tiles of the same keys stay on one XCD, by the same rule as prompts.
  int id = blockIdx.x, z = 0, tile = 0;
  if (a.splits > 1) {
    const int n = id / a.splits;
    z = id - n * a.splits;
    id = n;
  }
  if (a.row_tiles > 1) {
    if (units) {
      const int y = id >> 3, at = y / a.row_tiles;
      tile = y - at * a.row_tiles;
      id = (id & 7) + 8 * at;
      if (id >= units) return;
    } else {
      const int n = id / a.row_tiles;
      tile = id - n * a.row_tiles;
      id = n;
    }
  }
  const int s = a.n_seq > 1 ? id / a.kv_heads : 0, kv = id - s * a.kv_heads;
  const Sequence sq = sequence(a, s);
  const int n_rows = sq.nq * a.group;  // below 2^30: the host's check of max_q * group
  if (tile * 32 >= n_rows) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = tile * 32 + (lane & 31);
  const bool valid = row < n_rows;
  const int i = !valid ? 0 : a.group > 1 ? row / a.group : row, head = kv * a.group + (valid ? row - i * a.group : 0);
  const Seen me = valid ? seen(a, sq, i) : Seen{0, 0, 0};
  const int last = min(tile * 32 + 31, n_rows - 1) / a.group;
  const Range range = wave_range(a, sq, me, valid, tile * 32 / a.group, last);
  const Blocks<KB> blocks(sq.prefix, range.lo, range.hi, kBias == DistanceBias::None ? 0 : last + sq.nk - sq.nq);
  const int each = (blocks.count + a.splits - 1) / a.splits;
  const int j0 = min(blocks.count, z * each), j1 = min(blocks.count, j0 + each);

  const T* K = static_cast<const T*>(a.k) + sq.k0 * a.k_row + kv * a.k_head;
  const T* V = static_cast<const T*>(a.v) + sq.k0 * a.v_row + kv * a.v_head;

  constexpr int CH = KB * kChunks / 64, step = 64 / kChunks;
  const int r0 = lane / kChunks, c0 = lane % kChunks;
  unsigned at_k[CH], at_v[CH];
#pragma unroll
  for (int m = 0; m < CH; ++m) {
    const int r = r0 + m * step, ck = c0 ^ Block<D>::k_swizzle(r), cv = c0 ^ Block<D>::v_swizzle(r);
    at_k[m] = ck * 8 < a.dim ? 2u * static_cast<unsigned>(r) * static_cast<unsigned>(a.k_row) + 16u * ck : kNoChunk;
    at_v[m] = cv * 8 < a.dim ? 2u * static_cast<unsigned>(r) * static_cast<unsigned>(a.v_row) + 16u * cv : kNoChunk;
  }
  const Source<KB> from_k(K, a.k_row, sq.nk, a.dim), from_v(V, a.v_row, sq.nk, a.dim);
  const unsigned mine = wave * static_cast<unsigned>(kPlace * sizeof(T));
  const unsigned lds_k = lds_address(lds) + mine, lds_v = lds_k + KB * P * sizeof(T);
  // A wave's LDS reads of a block are done before loads overwrite it.
  auto load = [&](const Source<KB>& from, const unsigned (&at)[CH], unsigned to, int key) __attribute__((always_inline)) {
    const i32x4 r = from.resource(key, sq.nk);
    __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0_keep_vm());
    asm volatile("" ::: "memory");
#pragma unroll
    for (int m = 0; m < CH; ++m) lds_load16_buffer<true>(r, at[m], 0u, to + m * 1024u);
  };

  int j = j0 + wave, key0 = blocks.taken(j);
  if (j < j1) load(from_k, at_k, lds_k, key0);
  R rows;
  rows.start(lane);
  rows.load_q(static_cast<const T*>(a.q) + (sq.q0 + i) * a.q_row + head * a.q_head, a.dim, valid);
  rows.lo = me.lo;
  rows.hi = me.hi;
  rows.prefix = sq.prefix;
  rows.position = me.position;
  rows.slope = kBias == DistanceBias::Slopes ? -a.slopes[head] * a.per_unit : 0.f;
  const float* table = kBias == DistanceBias::Table ? a.table + static_cast<size_t>(head) * (2 * a.span + 1) + a.span : nullptr;
  if (j < j1) load(from_v, at_v, lds_v, key0);
  for (; j < j1; j += NW) {
    const int key = key0;
    const bool more = j + NW < j1;
    f32x16 t[1];
    T8 p[2];
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_only(CH));  // all but this block's V
    asm volatile("" ::: "memory");
    rows.scores((LdsBytes)(lds), mine, t);
    if (more) {
      key0 = blocks.taken(j + NW);
      load(from_k, at_k, lds_k, key0);
    }
    const typename R::Shift shift = rows.change(a, t, key, table, 0);
    if (!(key + KB <= sq.prefix || (key >= range.all_lo && key + KB <= range.all_hi))) rows.hide(t, key);
    if (j < j0 + NW) rows.open(a, t, shift);
    rows.total += rows.weigh_step(a, t, p, shift);
    if (more) __builtin_amdgcn_s_waitcnt(waitcnt_vm_only(CH));  // all but the next block's K
    else __builtin_amdgcn_s_waitcnt(waitcnt_vm_only(0));
    asm volatile("" ::: "memory");
    rows.weigh((LdsBytes)(lds) + KB * P * 2, mine, p);
    if (more) load(from_v, at_v, lds_v, key0);
  }

  // The waves' sums join: sum_w 2^(m_w - M) O_w and sum_w 2^(m_w - M) l_w.
  if (tid < 32) s_bad[tid] = 0;
  __syncthreads();  // every wave is done with its stages
  float* so = reinterpret_cast<float*>(lds);
  {
    const float total = halves_sum(rows.total);
    const unsigned bad = rows.doubtful(total);
    if (rows.g == 0) {
      s_reference[wave][lane & 31] = rows.reference;
      s_total[wave][lane & 31] = total;
      if (valid && (bad >> lane & 1)) s_bad[lane] = 1;  // every writer writes 1
    }
    float* mine = so + (wave * 32 + (lane & 31)) * OP + 4 * rows.g;
    if (valid) {
#pragma unroll
      for (int d = 0; d < R::DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          *reinterpret_cast<f32x4*>(mine + 32 * d + 2 * r) = f32x4{rows.o[d][r], rows.o[d][r + 1], rows.o[d][r + 2], rows.o[d][r + 3]};
    }
  }
  __syncthreads();
  const long long slot = ((static_cast<long long>(s) * a.kv_heads + kv) * a.row_tiles + tile) * a.splits + z;
  float* part = a.parts + slot * 32 * a.dim;
  float* ml = a.parts + static_cast<long long>(a.n_seq) * a.kv_heads * a.row_tiles * a.splits * 32 * a.dim + slot * 64;
  T* out = static_cast<T*>(a.out);
  const int mr = tid % 32, orow = tile * 32 + mr;  // NT is a multiple of 32: a thread's quads are of one row
  if (orow < n_rows && !s_bad[mr]) {
    float m = kNothing;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, s_reference[w][mr]);
    float wt[NW], total = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      wt[w] = __builtin_amdgcn_exp2f(s_reference[w][mr] - m);
      total += wt[w] * s_total[w][mr];
    }
    const int oi = orow / a.group, oh = kv * a.group + orow - oi * a.group;
    T* to = out + (sq.q0 + oi) * a.out_row + oh * a.out_head;
    const float inv = a.splits > 1 ? 1.f : total == 0.f ? 0.f : 1.0f / total;
    for (int d = tid / 32 * 4; d < a.dim; d += NT / 32 * 4) {
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(so + (w * 32 + mr) * OP + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(wt[w], x[e], v[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= inv;
      if (a.splits > 1) {
        *reinterpret_cast<f32x4*>(part + mr * a.dim + d) = v;
      } else {
        T4 h;
#pragma unroll
        for (int x = 0; x < 4; ++x) h[x] = to_half<T>(v[x]);
        *reinterpret_cast<T4*>(to + d) = h;
      }
    }
    if (a.splits > 1 && tid < 32) {
      ml[2 * mr] = m;
      ml[2 * mr + 1] = total;
    }
  }
  unsigned bad = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(s_bad[lane & 31] != 0));
  while (bad) {
    const int b = __builtin_ctz(bad);
    bad &= bad - 1;
    if (b % NW != wave) continue;
    const int orow = tile * 32 + b, oi = orow / a.group, oh = kv * a.group + orow - oi * a.group;
    const Seen m = seen(a, sq, oi);
    CarefulRow<T, D, KB, kCap, kBias> c;
    c.run(a, static_cast<const T*>(a.q) + (sq.q0 + oi) * a.q_row + oh * a.q_head, K, V, sq.nk, m.position, m.lo, m.hi, sq.prefix,
          kBias == DistanceBias::Slopes ? -a.slopes[oh] * a.per_unit : 0.f,
          a.table ? a.table + static_cast<size_t>(oh) * (2 * a.span + 1) + a.span : nullptr, blocks, j0, j1, lane);
    const float n = c.total == 0.f ? 0.f : 1.0f / c.total;
#pragma unroll
    for (int x = 0; x < c.ND; ++x) {
      const int d = lane + 64 * x;
      if (d >= a.dim) continue;
      if (a.splits > 1) part[b * a.dim + d] = c.sum[x];
      else out[(sq.q0 + oi) * a.out_row + oh * a.out_head + d] = to_half<T>(c.sum[x] * n);
    }
    if (a.splits > 1 && lane == 0) {
      ml[2 * b] = c.reference;
      ml[2 * b + 1] = c.total;
    }
  }
}

template <typename T, int D, bool kCap, DistanceBias kBias, int NW>
hipError_t launch_prompt(const AttendArgs& a, hipStream_t stream) {
  const int tiles = (a.max_q + 32 * NW - 1) / (32 * NW);
  const long long pairs = static_cast<long long>(a.n_seq) * a.heads, shared = static_cast<long long>(a.n_seq) * a.kv_heads;
  // Heads that share keys on one XCD, or each head, where that leaves no XCD more than a seventh above the mean; else every
  // tile for itself.
  const auto even = [](long long n) { return (n + 7) / 8 * 56 <= n * 8; };
  const int unit = even(shared) ? a.group : even(pairs) ? 1 : 0;
  const long long units = unit ? pairs / unit : pairs;
  const long long grid = unit ? (units + 7) / 8 * 8 * unit * tiles : pairs * tiles;
  LAYA_LAUNCH((attend_kernel<T, D, kCap, kBias, NW>), dim3(static_cast<unsigned>(grid)), dim3(64 * NW),
              kBias == DistanceBias::Table ? (2 * (a.span + kPad) + 1) * sizeof(float) : 0, stream, a, tiles, unit,
              static_cast<int>(units));
  return hipGetLastError();
}

template <typename T, int D, bool kCap, DistanceBias kBias>
hipError_t launch_kind(const AttendArgs& a, bool split, hipStream_t stream) {
  if (split) {
    const FewGrid grid = few_grid(a, a.row_tiles, a.splits);
    LAYA_LAUNCH((attend_split_kernel<T, D, kCap, kBias>), dim3(static_cast<unsigned>(grid.groups)), dim3(64 * split_waves<D>()), 0, stream, a, grid.units);
    return hipGetLastError();
  }
  // Eight waves take half the loads of four, but share one barrier on a CU.  Above 128 LDS holds one workgroup, and they are two a SIMD
  // instead of one (4 x 4,096 causal tokens of 16 heads of 256 865 and 529 us, of 192 786 and 421).  Below they gain where K and V outgrow the caches (16,384
  // causal tokens of 8 heads of 128 562 and 522 us, 2 x 8,192 of 16 heads of 96 437 and 396) and for heads of 80 and 96 at any length
  // (1,571 tokens 187 and 169), and lose where rows are few or ragged (32 of up to 2,000 of 128 291 and 307, 2,048 of 32 heads 57 and 64).
  if constexpr (D > 128) return launch_prompt<T, D, kCap, kBias, 8>(a, stream);
  if constexpr (D == 96 || D == 128) {
    const long long tiles8 = (a.max_q + 255) / 256 * static_cast<long long>(a.n_seq) * a.heads;
    if (tiles8 >= 2 * kPlannedUnits && (D == 96 || a.max_q >= 4096)) return launch_prompt<T, D, kCap, kBias, 8>(a, stream);
  }
  if constexpr (D <= 128) return launch_prompt<T, D, kCap, kBias, 4>(a, stream);
}

template <typename T, int D>
hipError_t launch_type(const AttendArgs& a, DistanceBias bias, bool cap, bool split, hipStream_t stream) {
  switch (bias) {
    case DistanceBias::None:
      return cap ? launch_kind<T, D, true, DistanceBias::None>(a, split, stream) : launch_kind<T, D, false, DistanceBias::None>(a, split, stream);
    case DistanceBias::Slopes:
      return cap ? launch_kind<T, D, true, DistanceBias::Slopes>(a, split, stream)
                 : launch_kind<T, D, false, DistanceBias::Slopes>(a, split, stream);
    default:
      return cap ? launch_kind<T, D, true, DistanceBias::Table>(a, split, stream)
                 : launch_kind<T, D, false, DistanceBias::Table>(a, split, stream);
  }
}

}  // namespace

template <>
hipError_t launch_attend_dim<LAYA_ATTEND_DIM>(const AttendArgs& a, DType t, DistanceBias bias, bool cap, bool split, hipStream_t stream) {
  return t == DType::F16 ? launch_type<f16, LAYA_ATTEND_DIM>(a, bias, cap, split, stream)
                         : launch_type<bf16, LAYA_ATTEND_DIM>(a, bias, cap, split, stream);
}

#else  // what is no kernel of a width

template <> hipError_t launch_attend_dim<64>(const AttendArgs&, DType, DistanceBias, bool, bool, hipStream_t);
template <> hipError_t launch_attend_dim<96>(const AttendArgs&, DType, DistanceBias, bool, bool, hipStream_t);
template <> hipError_t launch_attend_dim<128>(const AttendArgs&, DType, DistanceBias, bool, bool, hipStream_t);
template <> hipError_t launch_attend_dim<160>(const AttendArgs&, DType, DistanceBias, bool, bool, hipStream_t);
template <> hipError_t launch_attend_dim<192>(const AttendArgs&, DType, DistanceBias, bool, bool, hipStream_t);
template <> hipError_t launch_attend_dim<256>(const AttendArgs&, DType, DistanceBias, bool, bool, hipStream_t);

namespace {

// A row's sums over the splits: weights 2^(m_z - M), then one division.  4 us for 128 rows of 8 splits and 23 in a loop of dependent
// loads.  A workgroup a row: its four waves share the splits, in a
// fixed order, a lane four dims; every load of a wave is on its way before the first sum.
constexpr int kJoinWaves = 4, kJoinLoads = kMaxSplits / kJoinWaves;
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void join_kernel(AttendArgs a, int used) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x / used, r = blockIdx.x - tile * used;  // used: rows of a tile that any sequence has
  const int per = a.kv_heads * a.row_tiles, tiles = a.n_seq * per;  // below 2^24
  const int s = tile / per, w = tile - s * per;
  const int kv = w / a.row_tiles, row = (w - kv * a.row_tiles) * 32 + r;
  const int i = row / a.group;
  const int q0 = a.q_starts[s], nq = a.q_lengths[s];
  if (q0 < 0 || q0 >= a.q_rows || i >= min(min(nq, a.max_q), a.q_rows - q0)) return;
  const float* parts = a.parts + static_cast<long long>(tile) * a.splits * 32 * a.dim + r * a.dim;
  const float2* ml = reinterpret_cast<const float2*>(a.parts + static_cast<long long>(tiles) * a.splits * 32 * a.dim) +
                     static_cast<long long>(tile) * a.splits * 32 + r;
  float m = kNothing, l = 0.f;
  if (lane < a.splits) {
    const float2 x = ml[lane * 32];
    m = x.x;
    l = x.y;
  }
  const bool mine = 4 * lane < a.dim;
  f32x4 v[kJoinLoads];
#pragma unroll
  for (int n = 0; n < kJoinLoads; ++n) {
    const int z = wave + kJoinWaves * n;
    v[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (z < a.splits && mine) v[n] = *reinterpret_cast<const f32x4*>(parts + static_cast<long long>(z) * 32 * a.dim + 4 * lane);
  }
  const float top = wave_max(m);
  const float weight = __builtin_amdgcn_exp2f(m - top);
  const float total = wave_sum(weight * l);
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < kJoinLoads; ++n) {
    const float f = __shfl(weight, wave + kJoinWaves * n, kWave);
    if (wave + kJoinWaves * n < a.splits) {
#pragma unroll
      for (int x = 0; x < 4; ++x) sum[x] = __builtin_fmaf(f, v[n][x], sum[x]);
    }
  }
  __shared__ f32x4 others[kJoinWaves - 1][64];
  if (wave) others[wave - 1][lane] = sum;
  __syncthreads();
  if (wave || !mine) return;
#pragma unroll
  for (int n = 0; n < kJoinWaves - 1; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) sum[x] += others[n][lane][x];
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  typename Vec4<T>::type h;
#pragma unroll
  for (int x = 0; x < 4; ++x) h[x] = to_half<T>(sum[x] * inv);
  T* out = static_cast<T*>(a.out) + (q0 + i) * a.out_row + (kv * a.group + row - i * a.group) * a.out_head;
  *reinterpret_cast<typename Vec4<T>::type*>(out + 4 * lane) = h;
}

// The run of equal ids around each row of a sequence, a wave for 64 rows.  Where ids change comes from one ballot.  What begins before
// those rows or ends behind them is looked for from there, 512 rows at a time (kOpen false): one launch, but where one document
// fills a sequence of n rows its n / 64 waves take n / 512 steps each.  Or it is left open (kOpen true) for the two kernels below,
// so that each row is read and written a fixed number of times.  65,536 rows, documents of 200 and documents that fill their sequences, looked
// for and left open: in sequences of 1,024 4.4 and 4.8 us, 8.4 and 8.5; of 4,096 4.6 and 10.7, 8.6 and 8.5; of 16,384 4.5 and 34.7, 9.0 and 9.0;
// in one 4.6 and 130, 12.3 and 12.3.  One document of 2^20 rows 117 us, of 2^24 2.1 ms.
struct Run {
  int start, n;  // of a sequence, cut to the array
};
__device__ __forceinline__ Run run_of(const BoundsArgs& a, int s) {
  const int start = __builtin_amdgcn_readfirstlane(a.starts[s]), n = __builtin_amdgcn_readfirstlane(a.lengths[s]);
  return {start, start < 0 || start >= a.rows ? 0 : max(0, min(min(n, a.max_length), a.rows - start))};
}
constexpr int kLookedFor = 4096;  // rows of the longest sequences whose runs are looked for
constexpr int kOpenFirst = -1, kOpenEnd = INT_MAX;  // a run that begins, or ends, outside its 64 rows

template <bool kOpen>
__global__ __launch_bounds__(256) void document_bounds_kernel(BoundsArgs a, int groups) {
  const int lane = threadIdx.x & 63;
  const Run run = run_of(a, blockIdx.x / groups);
  const int n = run.n;
  const int i0 = (static_cast<int>(blockIdx.x % groups) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 64;
  if (i0 >= n) return;
  const int32_t* ids = a.documents + run.start;
  const int i = i0 + lane, last = min(n, i0 + 64) - 1;
  const int mine = ids[min(i, n - 1)], before = ids[max(0, min(i, n - 1) - 1)];
  const unsigned long long begins = __builtin_amdgcn_ballot_w64(i < n && (i == 0 || mine != before));
  // First row of the run that row i0 lies in, and the end of the one that row `last` lies in.
  int first = kOpenFirst, end = kOpenEnd;
  if constexpr (kOpen) {
    if (last + 1 == n || ids[last + 1] != ids[last]) end = last + 1;
  } else {
    if (!(begins & 1)) {
      const int id = __builtin_amdgcn_readfirstlane(mine);
      for (first = 0;;) {  // ends where a row differs, or before row 0
        int found = -1;
        const int from = i0 - 1 - first;  // rows above it are of the run
        for (int c = 7; c >= 0; --c) {
          const int at = from - 64 * c - lane;
          const unsigned long long other = __builtin_amdgcn_ballot_w64(at < 0 || ids[max(at, 0)] != id);
          if (other) found = 64 * c + __builtin_ctzll(other);
        }
        if (found >= 0) {
          first = from - found + 1;
          break;
        }
        first += 512;
      }
    }
    const int id = __builtin_amdgcn_readfirstlane(ids[last]);
    for (int gone = 0;; gone += 512) {
      int found = -1;
      for (int c = 7; c >= 0; --c) {
        const int at = last + 1 + gone + 64 * c + lane;
        const unsigned long long other = __builtin_amdgcn_ballot_w64(at >= n || ids[min(at, n - 1)] != id);
        if (other) found = 64 * c + __builtin_ctzll(other);
      }
      if (found >= 0) {
        end = last + 1 + gone + found;
        break;
      }
    }
  }
  if (i >= n) return;
  const unsigned long long upto = begins & (~0ull >> (63 - lane)), behind = lane == 63 ? 0 : begins >> (lane + 1);
  const int lo = upto ? i0 + 63 - __builtin_clzll(upto) : first;
  const int hi = behind ? i + 1 + __builtin_ctzll(behind) : end;
  a.bounds[run.start + i] = make_int2(lo, hi);
}

// Over a workgroup, in the order of its threads: the largest of what threads before this one hold, and of what all hold.
constexpr int kCarryThreads = 1024;
__device__ __forceinline__ int2 largest_before(int v) {
  __shared__ int waves[kCarryThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int by = 1; by < 64; by *= 2) {
    const int other = __shfl_up(v, by, kWave);
    if (lane >= by) v = max(v, other);
  }
  if (lane == 63) waves[wave] = v;
  const int own = __shfl_up(v, 1, kWave);
  __syncthreads();
  int before = INT_MIN, all = INT_MIN;
  for (int w = 0; w < kCarryThreads / 64; ++w) {
    if (w < wave) before = max(before, waves[w]);
    all = max(all, waves[w]);
  }
  __syncthreads();
  return make_int2(lane ? max(before, own) : before, all);
}

// What is open goes from each 64 rows to the next: a workgroup a sequence, 65,536 rows a step.  A group's last row has the first row
// of the run that leaves it (open: as the group before), so the run that enters a group begins at the largest such row before it; ends
// likewise, from the back, as negated rows.  The group's first row takes the one, its last row the other.
__global__ __launch_bounds__(kCarryThreads) void document_carry_kernel(BoundsArgs a) {
  const Run run = run_of(a, blockIdx.x);
  int2* bounds = a.bounds + run.start;
  const int groups = (run.n + 63) / 64;
  int first = kOpenFirst;
  for (int base = 0; base < groups; base += kCarryThreads) {
    const int g = base + threadIdx.x, at = 64 * g;
    const int2 r = largest_before(g < groups ? bounds[min(at + 63, run.n - 1)].x : kOpenFirst);
    if (g < groups && bounds[at].x == kOpenFirst) bounds[at].x = max(first, r.x);
    first = max(first, r.y);
  }
  int end = -kOpenEnd;
  for (int base = 0; base < groups; base += kCarryThreads) {
    const int g = groups - 1 - base - static_cast<int>(threadIdx.x), at = 64 * g;
    const int2 r = largest_before(g >= 0 ? -bounds[at].y : -kOpenEnd);
    const int last = min(at + 63, run.n - 1);
    if (g >= 0 && bounds[last].y == kOpenEnd) bounds[last].y = -max(end, r.x);
    end = max(end, r.y);
  }
}

__global__ __launch_bounds__(256) void document_fill_kernel(BoundsArgs a, int groups) {
  const int lane = threadIdx.x & 63;
  const Run run = run_of(a, blockIdx.x / groups);
  const int i0 = (static_cast<int>(blockIdx.x % groups) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 64;
  if (i0 >= run.n) return;
  const int rows = min(64, run.n - i0);
  int2* row = a.bounds + run.start + i0 + min(lane, rows - 1);
  const int2 mine = *row;
  const int first = __builtin_amdgcn_readfirstlane(mine.x), end = __builtin_amdgcn_readlane(mine.y, rows - 1);
  if (lane < rows && (mine.x == kOpenFirst || mine.y == kOpenEnd))
    *row = make_int2(mine.x == kOpenFirst ? first : mine.x, mine.y == kOpenEnd ? end : mine.y);
}

}  // namespace

hipError_t launch_attend(const AttendArgs& args, DType t, DistanceBias bias, bool cap, const AttendPlan& plan, hipStream_t stream) {
  AttendArgs a = args;
  a.row_tiles = plan.row_tiles;
  a.splits = plan.splits;
  const hipError_t e = a.dim <= 64    ? launch_attend_dim<64>(a, t, bias, cap, plan.split, stream)
                       : a.dim <= 96  ? launch_attend_dim<96>(a, t, bias, cap, plan.split, stream)
                       : a.dim <= 128 ? launch_attend_dim<128>(a, t, bias, cap, plan.split, stream)
                       : a.dim <= 160 ? launch_attend_dim<160>(a, t, bias, cap, plan.split, stream)
                       : a.dim <= 192 ? launch_attend_dim<192>(a, t, bias, cap, plan.split, stream)
                                      : launch_attend_dim<256>(a, t, bias, cap, plan.split, stream);
  if (e != hipSuccess || plan.splits <= 1) return e;
  const int used = a.row_tiles > 1 ? 32 : a.max_q * a.group;
  const dim3 grid(static_cast<unsigned>(static_cast<long long>(a.n_seq) * a.kv_heads * a.row_tiles * used));
  if (t == DType::F16) LAYA_LAUNCH(join_kernel<f16>, grid, dim3(64 * kJoinWaves), 0, stream, a, used);
  else LAYA_LAUNCH(join_kernel<bf16>, grid, dim3(64 * kJoinWaves), 0, stream, a, used);
  return hipGetLastError();
}

hipError_t launch_document_bounds(const BoundsArgs& a, hipStream_t stream) {
  const int groups = (a.max_length + 255) / 256;
  const dim3 grid(static_cast<unsigned>(static_cast<long long>(groups) * a.n_seq));
  if (a.max_length <= kLookedFor) {
    LAYA_LAUNCH(document_bounds_kernel<false>, grid, dim3(256), 0, stream, a, groups);
  } else {
    LAYA_LAUNCH(document_bounds_kernel<true>, grid, dim3(256), 0, stream, a, groups);
    LAYA_LAUNCH(document_carry_kernel, dim3(a.n_seq), dim3(kCarryThreads), 0, stream, a);
    LAYA_LAUNCH(document_fill_kernel, grid, dim3(256), 0, stream, a, groups);
  }
  return hipGetLastError();
}

#endif

}  // namespace laya
