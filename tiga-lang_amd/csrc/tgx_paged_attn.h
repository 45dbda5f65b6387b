// Attention over a paged relation: the kernels of tgx_paged.hip (16- and 32-bit
// caches) and tgx_paged_scaled.hip (caches in 8 bits).
//
// Dot-product attention of the newest tokens of each sequence over its pages
// of a key-value cache (Graph.paged):
//
//   out[r, h, g] = sum_j w_j v[slot(j), h],  w = softmax_j(scale q[r, h, g] . k[slot(j), h])
//
// over the positions j < length - (queries - 1 - t) of sequence b, r = b *
// queries + t; slot(j) = table[j / page_size] * page_size + j % page_size.
// `group` query heads share a key head.  A position whose page id names no
// page holds no key; a row that sees no key is zero.  A row's masked keys
// and values never reach it, whatever they hold.
//
// With a window W and S sinks (WIN) a row that sees the positions below
// `limit` sees those of them at limit - W or later, or below S.  The tiles that no
// row of a sequence sees lie between the last sink's and the window's first:
// they are taken out before the keys are cut into pieces (Piece::at).
//
// A cache in 8 bits (CODE) holds codes that 16-bit floats hold exactly, and a
// scale for every `block` slots and head: a key's scale multiplies its score and
// a value's its weight, so the tiles multiply codes.
//
// Bound: a cached row has to be read once, 4 * D bytes a key and head at 16
// bits, against 4 * group * D operations a new token: memory, for any group a
// model has and few new tokens.  The matrix tiles (16 bits, D = 32, 64, 128) read it
// once for 128 queries of its key head; paged_rows_kernel, which takes every other
// width and fp32, once for each query.
//
// Work split.  Lengths are only known on the device, so the launch is sized
// from the host's bounds and every workgroup finds its piece itself: the keys
// of all sequences, in tiles of 64, are cut into pieces of at most `c` tiles,
// c at least min_tiles and just large enough for W pieces to cover them all;
// sequence b gets k_b = max(1, ceil(tiles_b / c)) pieces of equal size, W
// together where there are fewer than W / 2 sequences, W + n_seqs at most.  A
// sequence of one piece writes its output; of several, each piece writes its
// running maximum, sum and unnormalized output, which a second launch joins in
// piece order.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "tgx_codes.h"
#include "tgx_device.h"
#include "tgx_host.h"
#include "tgx_paged.h"
#include "tgx_profile.h"
#include "tgx_vals.h"

namespace tgx {

struct PagedArgs {
  PagedRel rel;
  const void* q;
  const void* k;
  const void* v;
  int64_t qs_row, qs_head, qs_group;   // element strides of q
  int64_t ks_slot, ks_table, ks_head;  // of k: slot, table head, head
  int64_t vs_slot, vs_table, vs_head;
  void* out;              // [rows, heads, group, D] contiguous
  float scale_log2;       // score scale * log2(e)
  int heads;              // key heads per table
  int group;              // query heads per key head
  int D;
  int pieces;             // W
  int2* meta;             // [n_seqs] first piece and pieces of a sequence; null: one piece each
  float* partial;         // [piece, head, query] (D + 2) floats: output, maximum (log2), sum
  int window, sinks;      // WIN: at most the positions a table holds
  const float* k_scales;  // CODE: [slots / block, table heads, heads]
  const float* v_scales;
  unsigned block;
  int min_tiles;          // tiles a piece has at least
  int held;               // key heads a workgroup of the tile kernels holds (Wave)
};

// How a launch is cut: W pieces wanted, pieces launched at most, and whether
// any sequence can have several.
struct Cut {
  int64_t wanted, launched;
  bool split;
  int heads_held = 1;   // adjacent key heads of a workgroup (PagedArgs::held)
  int min_tiles = 4;    // tiles a piece has at least, where the sequence has them
};

// The launches over caches in 8 bits (tgx_paged_scaled.hip), without the join.
int paged_attn_scaled(const PagedArgs& a, const Cut& cut, int held, int dtype, int code,
                      hipStream_t stream);

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;       // keys a tile
constexpr int kMinTiles = 4;    // tiles that four waves of one head share at least

// 2^x on the hardware unit: exact 0 for -inf.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// What a windowed sequence of `length` tokens leaves out: the tiles from
// `sinks` on, `skip` of them (0: none).
struct Skipped {
  int sinks, skip;
};
__device__ __forceinline__ Skipped skipped_tiles(const PagedArgs& a, int length) {
  const int from = max(length - (a.rel.queries - 1), 0) - a.window;   // the oldest asking token's
  const int sinks = (min(a.sinks, length) + kTile - 1) / kTile;
  return Skipped{sinks, max(max(from, 0) / kTile - sinks, 0)};
}

// Tiles of a sequence of `length` tokens that some row sees.
template <bool WIN>
__device__ __forceinline__ int seen_tiles(const PagedArgs& a, int length) {
  const int n = (length + kTile - 1) / kTile;
  return WIN ? n - skipped_tiles(a, length).skip : n;
}

struct Piece {
  int seq;        // -1: no such piece
  int length;     // cached tokens of the sequence
  int index;      // piece of the sequence
  int count;      // pieces of the sequence
  int tile0, tile1;   // counted over the tiles that are seen
  Skipped gap;        // WIN
  // Where the seen tile (or, with `per` steps a tile, step) `v` lies.
  __device__ __forceinline__ int at(int v, int per) const {
    return v < gap.sinks * per ? v : v + gap.skip * per;
  }
};

// Positions that a row sees: below limit, and from `from` on or below `sinks`.
template <bool WIN>
struct Sight {
  int limit, from, sinks;
  Sight() = default;
  __device__ __forceinline__ Sight(const PagedArgs& a, int lim)
      : limit(lim), from(WIN ? max(lim, 0) - a.window : 0), sinks(a.sinks) {}
  __device__ __forceinline__ bool operator()(int pos) const {
    return pos < limit && (!WIN || pos >= from || pos < sinks);
  }
  // Whether it sees all of the n positions from pos on, as every row between it
  // and `newest` does.
  __device__ __forceinline__ bool all(int pos, int n, const Sight& newest) const {
    return pos + n <= limit && (!WIN || pos >= newest.from || pos + n <= sinks);
  }
};

// Cuts n tiles into p.count pieces whose sizes differ by one at most.
__device__ __forceinline__ void cut_tiles(Piece& p, int n) {
  const int each = n / p.count, more = n % p.count;
  p.tile0 = p.index * each + min(p.index, more);
  p.tile1 = p.tile0 + each + (p.index < more);
}

// Piece `x` of the launch; every wave finds it by itself.  Lane l looks
// after the sequences [l, l + 1) * ceil(n / 64).
template <bool WIN>
__device__ __forceinline__ Piece find_piece(const PagedArgs& a, int x) {
  const PagedRel& r = a.rel;
  const int pieces = a.pieces;
  Piece p{-1, 0, 0, 1, 0, 0, {0, 0}};
  if (a.meta == nullptr) {   // one piece a sequence
    if (x >= r.n_seqs) return p;
    p.seq = x;
    p.length = paged_length(r, x);
    p.tile1 = seen_tiles<WIN>(a, p.length);
    if (WIN) p.gap = skipped_tiles(a, p.length);
    return p;
  }
  const int lane = lane_id();
  if (r.n_seqs == 1) {
    p.length = paged_length(r, 0);
    const int n = seen_tiles<WIN>(a, p.length);
    if (WIN) p.gap = skipped_tiles(a, p.length);
    const int c = max(a.min_tiles, (n + pieces - 1) / pieces);
    p.count = max(1, (n + c - 1) / c);
    if (x >= p.count) return p;
    p.seq = 0;
    p.index = x;
    cut_tiles(p, n);
    return p;
  }
  const int per = (r.n_seqs + 63) / 64;
  const int b0 = lane * per, b1 = min(r.n_seqs, b0 + per);
  int tiles = 0;
  for (int b = b0; b < b1; ++b) tiles += seen_tiles<WIN>(a, paged_length(r, b));
  const int total = read_lane(wave_prefix(tiles), 63);
  // Rounding up adds a piece a sequence at most, which are taken off first.
  const int room = max(pieces - r.n_seqs, (pieces + 1) / 2);
  const int c = max(a.min_tiles, (total + room - 1) / room);
  int mine = 0;
  if (per == 1)
    mine = b0 < b1 ? max(1, (tiles + c - 1) / c) : 0;
  else
    for (int b = b0; b < b1; ++b)
      mine += max(1, (seen_tiles<WIN>(a, paged_length(r, b)) + c - 1) / c);
  const int end = wave_prefix(mine);
  const unsigned long long hit = __ballot(x < end && x >= end - mine);
  if (!hit) return p;
  const int owner = __builtin_ctzll(hit);
  int at = end - mine, found = -1, k = 1, n = 0, len = 0;
  for (int b = b0; b < b1 && found < 0; ++b) {
    len = paged_length(r, b);
    n = seen_tiles<WIN>(a, len);
    k = max(1, (n + c - 1) / c);
    if (x < at + k) found = b;
    else at += k;
  }
  p.seq = read_lane(found, owner);
  p.length = read_lane(len, owner);
  p.count = read_lane(k, owner);
  p.index = x - read_lane(at, owner);
  cut_tiles(p, read_lane(n, owner));
  if (WIN) p.gap = skipped_tiles(a, p.length);
  return p;
}

// Running maximum (log2 units), sum and weighted sum of 8 values per lane.
struct State8 {
  float m, l, acc[8];
  __device__ __forceinline__ void init() {
    m = kNegInf;
    l = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
  }
  __device__ __forceinline__ void merge(float m2, float l2, const float (&a2)[8]) {
    const float mn = fmaxf(m, m2);
    // (A maximum of -inf has no weight; +inf against itself is the formula's NaN.)
    const float a = m == kNegInf ? 0.f : exp2_hw(m - mn);
    const float b = m2 == kNegInf ? 0.f : exp2_hw(m2 - mn);
    l = l * a + l2 * b;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = acc[k] * a + a2[k] * b;
    m = mn;
  }
  __device__ __forceinline__ void merge_xor(int mask) {
    float a2[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) a2[k] = __shfl_xor(acc[k], mask, 64);
    merge(__shfl_xor(m, mask, 64), __shfl_xor(l, mask, 64), a2);
  }
};

// One workgroup per (piece, head, query): LPK lanes hold a row of D values, 8
// each, and a wave's 64 / LPK lane groups take a key each; the states of the
// groups and the four waves are merged at the end.  A key head's queries read
// its rows one by one, from L2 where they meet there: 64 sequences of 100 to
// 4000 tokens, fp32, 8 heads of 128: 225 us with one query a head (4.9 TB/s),
// 663 us with four; bf16 with four, heads of 256 780 us, of 96 432 us.
template <int DT, int LPK, int CODE, bool WIN>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  using C = CacheVals<DT, CODE>;   // how k and v are held
  using CT = typename C::T;
  const PagedRel& r = a.rel;
  const int all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;   // queries of one (sequence, head)
  const unsigned item = blockIdx.x / static_cast<unsigned>(rows);
  const int row = static_cast<int>(blockIdx.x % static_cast<unsigned>(rows));
  const int head = static_cast<int>(item % static_cast<unsigned>(all_heads));
  const int x = static_cast<int>(item / static_cast<unsigned>(all_heads));
  const Piece p = find_piece<WIN>(a, x);
  if (p.seq < 0) return;
  const int th = head / a.heads, kh = head % a.heads;
  const int t = row / a.group, g = row % a.group;
  if (a.meta && p.index == 0 && row == 0 && head == 0 && threadIdx.x == 0)
    a.meta[p.seq] = make_int2(x, p.count);

  const int wave = threadIdx.x >> 6, lane = lane_id();
  const int part = lane % LPK, sub = lane / LPK;
  const bool has = 8 * part < a.D;
  const int64_t q_row = (static_cast<int64_t>(p.seq) * r.queries + t) * r.heads + th;
  float q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (has)
    V::unpack(V::load(static_cast<const T*>(a.q) + q_row * a.qs_row + kh * a.qs_head +
                      g * a.qs_group + 8 * part), q);
  const CT* kb = static_cast<const CT*>(a.k) + th * a.ks_table + kh * a.ks_head + 8 * part;
  const CT* vb = static_cast<const CT*>(a.v) + th * a.vs_table + kh * a.vs_head + 8 * part;
  const int32_t* table = r.table + p.seq * r.seq_stride + th * r.head_stride;

  const Sight<WIN> sees(a, p.length - (r.queries - 1 - t));
  const int last = WIN ? p.tile1 * kTile : min(sees.limit, p.tile1 * kTile);
  State8 s;
  s.init();
  for (int i = p.tile0 * kTile + wave * (64 / LPK) + sub; i < last; i += 4 * (64 / LPK)) {
    const int j = WIN ? p.at(i, kTile) : i;
    if (WIN && !sees(j)) continue;
    const int slot = paged_slot(r, table, j);
    if (slot < 0) continue;
    float kv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float vv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (has) {
      const typename C::Raw kr = C::load(kb + slot * a.ks_slot);
      const typename C::Raw vr = C::load(vb + slot * a.vs_slot);
      C::unpack(kr, kv);
      C::unpack(vr, vv);
    }
    float scale = a.scale_log2;
    if constexpr (CODE != 0) {
      const unsigned block = static_cast<unsigned>(slot) / a.block;
      const int64_t at = static_cast<int64_t>(block) * all_heads + head;
      scale *= a.k_scales[at];
      const float vs = a.v_scales[at];
#pragma unroll
      for (int e = 0; e < 8; ++e) vv[e] *= vs;
    }
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) dot += q[e] * kv[e];
    s.merge(group_sum<LPK>(dot) * scale, 1.f, vv);
  }
#pragma unroll
  for (int mask = LPK; mask < 64; mask <<= 1) s.merge_xor(mask);

  __shared__ float ml[4][2];
  __shared__ float acc[4][8 * LPK];
  if (sub == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[wave][8 * part + i] = s.acc[i];
    if (part == 0) {
      ml[wave][0] = s.m;
      ml[wave][1] = s.l;
    }
  }
  __syncthreads();
  if (wave != 0 || sub != 0 || !has) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = acc[w][8 * part + i];
    s.merge(ml[w][0], ml[w][1], o);
  }
  if (p.count == 1) {
    const float inv = s.l == 0.f ? 0.f : 1.f / s.l;
#pragma unroll
    for (int i = 0; i < 8; ++i) s.acc[i] *= inv;
    V::store(static_cast<T*>(a.out) + ((q_row * a.heads + kh) * a.group + g) * a.D + 8 * part,
             s.acc);
  } else {
    float* dst = a.partial +
                 ((static_cast<int64_t>(x) * all_heads + head) * rows + row) * (a.D + 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[8 * part + i] = s.acc[i];
    if (part == 0) {
      dst[a.D] = s.m;
      dst[a.D + 1] = s.l;
    }
  }
}

// ---------------------------------------------------------------------------
// Matrix tiles (bf16, fp16; D = 32, 64, 128)
//
// With lane l, g = l / 16, lr = l % 16 (v_mfma_f32_16x16x32, as in the dense
// tiles): S^T = K Q^T of 16 queries takes K fragments of 16 bytes a lane, 64
// contiguous bytes of each of 16 rows; the lane's results are four keys of
// one query for each 16 keys, which is P^T as the B operand of O^T = V^T P^T
// under the key order {4g .. 4g + 3, 16 + 4g ..}; V^T is read down the columns
// of a V tile staged in LDS (ds_read_b64_tr_b16).  A weight is multiplied as
// the sum of two 16-bit values, so that only the output's rounding is left.
// Up to 64 queries the matrix unit has the time to spare (at D = 128, 24
// instructions of 16 cycles for the 16 KB of 32 keys, which take some 700
// cycles of a CU's share of memory).  Above it is the bound, and the second
// part is kept all the same, so that a row's accuracy does not depend on how
// many ask: 512 new tokens of four sequences of 3000 to 4000, 8 x 4 heads of
// 128, bf16, take 283 us (400 TFLOP/s), 231 us with one part.
//
// Two kernels.  Up to 16 queries of one (sequence, head): paged_tile_kernel,
// whose four waves run through every fourth step of KEYS keys by themselves
// with no barrier before the end.  More: paged_block_kernel, whose waves take
// 16 queries each of tiles of 64 keys that all four stage together.

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
template <typename T>
struct Frag;
template <>
struct Frag<__bf16> {
  typedef bf16x8 v8;
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  static constexpr uint32_t kExponent = 0x7F80u;
  static constexpr float kRescaleLog2 = 8.f, kLiftLog2 = 0.f;
};
template <>
struct Frag<_Float16> {
  typedef f16x8 v8;
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  static constexpr uint32_t kExponent = 0x7C00u;
  static constexpr float kRescaleLog2 = 1.f, kLiftLog2 = 14.f;
};
template <typename T>
using vec8 = typename Frag<T>::v8;
template <typename T>
using vec4 = typename Frag<T>::v4;
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Max and sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float group4_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float group4_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// Row stride (elements) of a staged tile: free of bank conflicts as in the
// dense tiles.
template <int D>
constexpr int kRow = D == 128 ? 144 : D == 64 ? 80 : 48;

// The running maximum m only moves when a step's exceeds it by kRescaleLog2
// (log2 units), and a weight is 2^(s - m + kLiftLog2): a factor that the sum of
// the weights carries too.  fp16 has no numbers below 2^-24, so there the
// weights fill the range up to 2^15: their two parts are off by 2^-39 of the
// largest at most, a weight of e^-20 by 2^-10 of itself.  (Unlifted, those
// below 2^-25 = e^-17.3 are lost from the output and kept in the sum.)  It
// costs nothing: 24 sequences of up to 3000 tokens x 4, 16 heads of 64, 35.5 us.

// The lane's part of 16 queries: row `row` of the (sequence, head), its
// fragments, and the positions it sees (rows past the last see as the last).
// Fragment i holds eight values of a row: from 32 i + 8 g on, or (PAIRS) in the
// order in which the halves of 16 codes a lane meet them, 64 (i / 2) + 16 g + 8
// (i % 2).
template <typename T, int D, bool WIN, bool PAIRS = false>
struct Query {
  vec8<T> f[D / 32];
  Sight<WIN> sees;
  Query() = default;
  __device__ __forceinline__ Query(const PagedArgs& a, const Piece& p, int th, int kh, int row,
                                   int rows, int g) {
    const int t = min(row / a.group, a.rel.queries - 1), gq = row % a.group;
    sees = Sight<WIN>(a, p.length - (a.rel.queries - 1 - t));
    const int64_t q_row = (static_cast<int64_t>(p.seq) * a.rel.queries + t) * a.rel.heads + th;
    const T* q = static_cast<const T*>(a.q) + q_row * a.qs_row + kh * a.qs_head +
                 gq * a.qs_group;
#pragma unroll
    for (int kc = 0; kc < D / 32; ++kc) {
      const int d = PAIRS ? 64 * (kc / 2) + 16 * g + 8 * (kc % 2) : 32 * kc + 8 * g;
      f[kc] = row < rows ? *reinterpret_cast<const vec8<T>*>(q + d) : vec8<T>{};
    }
  }
};

// Scaled scores of 16 KT keys from position `pos` become weights 2^(s - m + lift)
// under the running maximum m; l and o follow it.  `gone`: bit k set, key k is
// not there; `masked`: some key may be hidden from the lane's query.
template <typename T, bool WIN, int KT, int DT>
__device__ __forceinline__ void weigh(f32x4 (&c)[KT], bool masked, unsigned long long gone,
                                      int pos, const Sight<WIN>& sees, int g, float& m, float& l,
                                      f32x4 (&o)[DT]) {
  if (masked) {
    gone >>= 4 * g;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((gone >> (16 * kt + i) & 1) || !sees(pos + 16 * kt + 4 * g + i)) c[kt][i] = kNegInf;
  }
  float top = kNegInf;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, c[kt][i]);
  top = group4_max(top);
  // (The difference, not the sum: m + 1 may round away from where m is large.)
  if (__any(top - m > Frag<T>::kRescaleLog2)) {
    const float mn = fmaxf(m, top);
    const float alpha = m == kNegInf ? 0.f : exp2_hw(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
  }
  const float mo = (m == kNegInf ? 0.f : m) - Frag<T>::kLiftLog2;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[kt][i] = exp2_hw(c[kt][i] - mo);
      l += c[kt][i];
    }
}

// o += V^T P^T over the 16 KT staged rows at `v`, for QT tiles of 16 queries.
template <typename T, int D, int KT, int QT>
__device__ __forceinline__ void add_values(const T* v, const f32x4 (&c)[QT][KT], int g, int lr,
                                           f32x4 (&o)[QT][D / 16]) {
  constexpr int ROW = kRow<D>;
#pragma unroll
  for (int k2 = 0; k2 < KT / 2; ++k2) {
    vec8<T> ph[QT], pl[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = c[qt][2 * k2 + j / 4][j % 4];
        ph[qt][j] = static_cast<T>(w);
        pl[qt][j] = static_cast<T>(w - static_cast<float>(ph[qt][j]));
      }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const T* src = v + (32 * k2 + 4 * g + (lr >> 2)) * ROW + 16 * dt + 4 * (lr & 3);
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(src));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(src + 16 * ROW));
      const u32x2 wl = __builtin_bit_cast(u32x2, lo), wh = __builtin_bit_cast(u32x2, hi);
      const vec8<T> vt = __builtin_bit_cast(vec8<T>, (u32x4{wl[0], wl[1], wh[0], wh[1]}));
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        o[qt][dt] = mfma(vt, ph[qt], o[qt][dt]);
        o[qt][dt] = mfma(vt, pl[qt], o[qt][dt]);
      }
    }
  }
}

// The same key by key (`weights`: the wave's [16 KT][16] floats of LDS), for
// steps that hold a NaN or Inf among their values: what a query does not see is
// left out, not multiplied by 0, and an Inf is weighed once, not by the two
// parts of its weight (Inf - Inf).
template <typename T, int D, bool WIN, int KT>
__device__ __forceinline__ void add_seen_values(const T* v, const f32x4 (&c)[KT], int g, int lr,
                                                int pos, const Sight<WIN>& sees, float* weights,
                                                f32x4 (&o)[D / 16]) {
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) weights[(16 * kt + 4 * g + i) * 16 + lr] = c[kt][i];
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  for (int key = 0; key < 16 * KT; ++key) {
    if (!sees(pos + key)) continue;
    const float w = weights[key * 16 + lr];
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const vec4<T> vv = *reinterpret_cast<const vec4<T>*>(v + key * kRow<D> + 16 * dt + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[dt][e] += w * static_cast<float>(vv[e]);
    }
  }
}

// Largest magnitudes (as bits) of the even and odd elements seen: an element
// is a NaN or Inf when its exponent is all ones.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <typename T>
struct Largest {
  u16x2 top = {0, 0};
  __device__ __forceinline__ void see(const vec8<T>& v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
  }
  __device__ __forceinline__ bool odd() const {
    return top[0] >= Frag<T>::kExponent || top[1] >= Frag<T>::kExponent;
  }
};

// The states of the WAVES waves that share 16 queries, joined in wave order and
// written: the output, or the piece's partial.  `smem` holds [group][wave][16][D
// + 4] outputs, then maxima and sums; row0 is the first group's first row.
template <typename T, int D, int WAVES>
__device__ __forceinline__ void join_waves(const PagedArgs& a, const Piece& p, int x, int head,
                                           int th, int kh, int row0, int apart, int rows,
                                           char* smem, float m, float l,
                                           const f32x4 (&o)[D / 16]) {
  constexpr int GROUPS = 4 / WAVES;
  float* jo = reinterpret_cast<float*>(smem);
  float* jm = jo + 4 * 16 * (D + 4);
  const int wave = threadIdx.x >> 6, lane = lane_id(), g = lane >> 4, lr = lane & 15;
  __syncthreads();
  const float sum_l = group4_sum(l);
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt)
    *reinterpret_cast<f32x4*>(jo + (wave * 16 + lr) * (D + 4) + 16 * dt + 4 * g) = o[dt];
  if (g == 0) {
    jm[2 * (wave * 16 + lr)] = m;
    jm[2 * (wave * 16 + lr) + 1] = sum_l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < GROUPS * 16 * (D / 4); i += 256) {
    const int qr = i / (D / 4), d = i % (D / 4) * 4, row = row0 + qr / 16 * apart + qr % 16;
    if (row >= rows) continue;
    const int at0 = qr / 16 * WAVES * 16 + qr % 16;
    float mw[WAVES], mx = kNegInf;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      mw[w] = jm[2 * (at0 + 16 * w)];
      mx = fmaxf(mx, mw[w]);
    }
    float sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      // (A wave without a maximum has no weight, or a NaN of its own.)
      const float f = mw[w] == kNegInf ? 1.f : exp2_hw(mw[w] - mx);
      sum += f * jm[2 * (at0 + 16 * w) + 1];
      acc += f * *reinterpret_cast<const f32x4*>(jo + (at0 + 16 * w) * (D + 4) + d);
    }
    if (p.count == 1) {
      const int t = row / a.group, gq = row % a.group;
      const int64_t q_row = (static_cast<int64_t>(p.seq) * a.rel.queries + t) * a.rel.heads + th;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      vec4<T> w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(acc[e] * inv);
      *reinterpret_cast<vec4<T>*>(static_cast<T*>(a.out) +
                                  ((q_row * a.heads + kh) * a.group + gq) * D + d) = w;
    } else {
      float* dst = a.partial +
                   ((static_cast<int64_t>(x) * a.rel.heads * a.heads + head) * rows + row) *
                       (D + 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[d + e] = acc[e];
      if (d == 0) {
        dst[D] = mx;
        dst[D + 1] = sum;
      }
    }
  }
}

// What a wave of a tile kernel does: workgroups of one piece hold a.held adjacent key
// heads each, of one table, with 4 / a.held waves a head that take its steps in turn.
// Adjacent heads lie side by side in a slot: together they are read in longer
// stretches, and a piece's heads on one XCD share its L2's lines (24 sequences of up to
// 3000 x 4 tokens, 16 heads of 64, 8 bits: 28.5 us with heads spread over XCDs, 20 us).
struct Wave {
  int x, head, th, kh;       // piece; head over all tables; table head and key head
  int group, part, parts;    // head of the workgroup; turn, of how many
  __device__ __forceinline__ Wave(const PagedArgs& a, int wave) {
    const unsigned heads = a.rel.heads * a.heads / static_cast<unsigned>(a.held);
    // A piece's heads are workgroups 8 apart, on one XCD.
    const unsigned of8 = blockIdx.x / 8u;
    x = static_cast<int>(of8 / heads * 8u + blockIdx.x % 8u);
    parts = 4 / a.held;
    group = wave / parts;
    part = wave % parts;
    head = static_cast<int>(of8 % heads) * a.held + group;
    th = head / a.heads;
    kh = head % a.heads;
  }
};

// join_waves for 16 queries of each of the workgroup's heads.
template <typename T, int D>
__device__ __forceinline__ void join_heads(const PagedArgs& a, const Piece& p, const Wave& wv,
                                           int rows, char* smem, float m, float l,
                                           const f32x4 (&o)[D / 16]) {
  float* jo = reinterpret_cast<float*>(smem);
  float* jm = jo + 4 * 16 * (D + 4);
  const int wave = threadIdx.x >> 6, lane = lane_id(), g = lane >> 4, lr = lane & 15;
  __syncthreads();
  const float sum_l = group4_sum(l);
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt)
    *reinterpret_cast<f32x4*>(jo + (wave * 16 + lr) * (D + 4) + 16 * dt + 4 * g) = o[dt];
  if (g == 0) {
    jm[2 * (wave * 16 + lr)] = m;
    jm[2 * (wave * 16 + lr) + 1] = sum_l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.held * 16 * (D / 4); i += 256) {
    const int group = i / (16 * (D / 4)), row = i / (D / 4) % 16, d = i % (D / 4) * 4;
    if (row >= rows) continue;
    const int at0 = group * wv.parts * 16 + row;
    float mx = kNegInf;
    for (int w = 0; w < wv.parts; ++w) mx = fmaxf(mx, jm[2 * (at0 + 16 * w)]);
    float sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < wv.parts; ++w) {
      // (A wave without a maximum has no weight, or a NaN of its own.)
      const float mw = jm[2 * (at0 + 16 * w)];
      const float f = mw == kNegInf ? 1.f : exp2_hw(mw - mx);
      sum += f * jm[2 * (at0 + 16 * w) + 1];
      acc += f * *reinterpret_cast<const f32x4*>(jo + (at0 + 16 * w) * (D + 4) + d);
    }
    const int head = wv.head - wv.group + group, kh = wv.kh - wv.group + group;
    if (p.count == 1) {
      const int t = row / a.group, gq = row % a.group;
      const int64_t q_row =
          (static_cast<int64_t>(p.seq) * a.rel.queries + t) * a.rel.heads + wv.th;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      vec4<T> w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(acc[e] * inv);
      *reinterpret_cast<vec4<T>*>(static_cast<T*>(a.out) +
                                  ((q_row * a.heads + kh) * a.group + gq) * D + d) = w;
    } else {
      float* dst = a.partial +
                   ((static_cast<int64_t>(wv.x) * a.rel.heads * a.heads + head) * rows + row) *
                       (D + 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[d + e] = acc[e];
      if (d == 0) {
        dst[D] = mx;
        dst[D + 1] = sum;
      }
    }
  }
}
template <int D>
constexpr size_t kJoinBytes = sizeof(float) * 4 * 16 * (D + 4 + 2);

// Up to 16 queries.  Memory is kept busy by order alone: a step's K loads are
// issued as soon as the step before has multiplied its own, its V loads as
// soon as the step before has staged its own, and the page ids one step ahead
// of that, so a wave always has 8 KB (D = 128) or more on its way.  Measured:
// four sequences of 100k to 131k, 8 x 4 heads of 128, 347 us (5.6 TB/s, of 6.3
// that plain reads reach); 64 of 100 to 4000 tokens 120 us (4.6 TB/s, the
// join among them).
//
// Keys a step: 64 leave room for fewer workgroups (24 sequences of up to 3000
// tokens, 16 heads of 64: 47 us, 37 us with 32).  Workgroups a CU: at D = 128
// three would need K's and V's fragments to share registers, and measured
// equal; at D = 64 four spill (42 us).
constexpr int KEYS = 32;
template <typename T, int D, bool WIN>
__global__ __launch_bounds__(256, (D == 128 ? 2 : D == 64 ? 3 : 4)) void paged_tile_kernel(
    PagedArgs a) {
  constexpr int KT = KEYS / 16, KC = D / 32, ROW = kRow<D>;
  constexpr size_t kStage = sizeof(T) * 4 * KEYS * ROW;
  constexpr size_t kBytes = kStage + sizeof(float) * 4 * KEYS * 16;
  __shared__ __align__(16) char smem[kBytes > kJoinBytes<D> ? kBytes : kJoinBytes<D>];
  const PagedRel& r = a.rel;
  const unsigned all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  Wave wv(a, wave);
  if (!WIN) {   // one head a workgroup, in order
    wv.head = static_cast<int>(blockIdx.x % all_heads);
    wv.x = static_cast<int>(blockIdx.x / all_heads);
    wv.th = wv.head / a.heads, wv.kh = wv.head % a.heads;
    wv.group = 0, wv.part = wave, wv.parts = 4;
  }
  const Piece p = find_piece<WIN>(a, wv.x);
  if (p.seq < 0) return;
  const int th = wv.th, kh = wv.kh, parts = wv.parts;
  if (a.meta && p.index == 0 && wv.head == 0 && threadIdx.x == 0)
    a.meta[p.seq] = make_int2(wv.x, p.count);

  const int g = lane >> 4, lr = lane & 15;
  const Query<T, D, WIN> q(a, p, th, kh, lr, rows, g);
  // What the oldest and the newest of the queries see, and the piece's end.
  const Sight<WIN> oldest(a, p.length - (r.queries - 1)), newest(a, p.length);
  const int high = WIN ? p.length : min(p.length, p.tile1 * kTile);
  const T* kb = static_cast<const T*>(a.k) + th * a.ks_table + kh * a.ks_head + 8 * g;
  const T* vb = static_cast<const T*>(a.v) + th * a.vs_table + kh * a.vs_head + 8 * g;
  const int32_t* table = r.table + p.seq * r.seq_stride + th * r.head_stride;
  // The wave's staged V, and its weights where they are taken key by key.
  T* stage = reinterpret_cast<T*>(smem) + wave * KEYS * ROW;
  float* weights = reinterpret_cast<float*>(smem + kStage) + wave * KEYS * 16;

  // Steps of this wave: first + parts i < last.  Lane l keeps the page id of key
  // l (mod KEYS) of a step.
  const int first = p.tile0 * (kTile / KEYS) + wv.part;
  constexpr int PER = kTile / KEYS;
  const int last = WIN ? min(p.tile1 * PER, (high + KEYS - 1) / KEYS - p.gap.skip * PER)
                       : (high + KEYS - 1) / KEYS;
  auto start = [&](int step) { return (WIN ? p.at(step, PER) : step) * KEYS; };
  auto page_id = [&](int step) {
    const int pos = min(start(step) + lane % KEYS, r.pages_per_seq * r.page_size - 1);
    return table[static_cast<unsigned>(pos) / static_cast<unsigned>(r.page_size)];
  };
  auto slot_of = [&](int step, int id) {
    const unsigned pos = start(step) + lane % KEYS;
    const bool there = static_cast<int>(pos) < high &&
                       (!WIN || (step < last && (static_cast<int>(pos) >= oldest.from ||
                                                 static_cast<int>(pos) < oldest.sinks))) &&
                       static_cast<unsigned>(id) < static_cast<unsigned>(r.num_pages);
    return there ? id * r.page_size + static_cast<int>(pos % static_cast<unsigned>(r.page_size))
                 : -1;
  };
  // (A key that is not there loads slot 0, and is masked.)
  auto load = [&](vec8<T>(&f)[KT][KC], const T* base, int64_t stride, int slot) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int s = max(__shfl(slot, 16 * kt + lr, 64), 0);
      const T* row = base + s * stride;
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) f[kt][kc] = *reinterpret_cast<const vec8<T>*>(row + 32 * kc);
    }
  };

  float m = kNegInf, l = 0.f;
  f32x4 o[1][D / 16];
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) o[0][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (first < last) {
    vec8<T> kf[KT][KC], vf[KT][KC];
    int slot = slot_of(first, page_id(first));
    load(kf, kb, a.ks_slot, slot);
    load(vf, vb, a.vs_slot, slot);
    int next_id = page_id(first + parts);
    for (int step = first; step < last; step += parts) {
      const int next = slot_of(step + parts, next_id);
      next_id = page_id(step + 2 * parts);
      const unsigned long long gone = __ballot(slot < 0);   // bit k: key k is not there
      f32x4 c[1][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) c[0][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kc = 0; kc < KC; ++kc)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) c[0][kt] = mfma(kf[kt][kc], q.f[kc], c[0][kt]);
      load(kf, kb, a.ks_slot, next);

      const int pos = start(step);
      const bool part = !oldest.all(pos, KEYS, newest);   // some query sees only a part
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) c[0][kt] *= a.scale_log2;
      weigh<T, WIN>(c[0], gone || part, gone, pos, q.sees, g, m, l, o[0]);

      // Stage V; a key that is not there counts as a row of zeros.
      if (gone) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
          if (gone >> (16 * kt + lr) & 1) {
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) vf[kt][kc] = vec8<T>{};
          }
      }
      Largest<T> largest;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) largest.see(vf[kt][kc]);
      const bool odd = __any(largest.odd());
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
          *reinterpret_cast<vec8<T>*>(stage + (16 * kt + lr) * ROW + 32 * kc + 8 * g) = vf[kt][kc];
      load(vf, vb, a.vs_slot, next);
      __builtin_amdgcn_wave_barrier();
      if (!odd)
        add_values<T, D, KT, 1>(stage, c, g, lr, o);
      else
        add_seen_values<T, D, WIN>(stage, c[0], g, lr, pos, q.sees, weights, o[0]);
      slot = next;
    }
  }
  if constexpr (WIN)
    join_heads<T, D>(a, p, wv, rows, smem, m, l, o[0]);
  else
    join_waves<T, D, 4>(a, p, wv.x, wv.head, th, kh, 0, 16, rows, smem, m, l, o[0]);
}

// More than 16 queries.  The four waves stage 64 keys together, the next tile's
// loads in flight in registers while this one is multiplied.  KW waves share
// 16 QT queries and take 64 / KW keys of a tile each, so a workgroup holds 64 QT
// / KW queries: 32 (KW = 2), 64, or 128 (QT = 2), the smallest that holds all
// of them (one read of the keys), 128 where none does.  Workgroups of the same
// keys are 8 apart, on one XCD's L2.
template <typename T, int D, int KW, int QT, int CODE, bool WIN>
__global__ __launch_bounds__(256, (D == 128 || QT == 2 ? 2 : 3)) void paged_block_kernel(
    PagedArgs a) {
  using VT = std::conditional_t<CODE == 0, T, __bf16>;   // of weights and values as multiplied
  using Raw = std::conditional_t<CODE == 0, vec8<T>, u32x2>;   // eight cached values
  using CT = std::conditional_t<CODE == 0, T, uint8_t>;
  constexpr int KT = 4 / KW, KC = D / 32, ROW = kRow<D>, QUERIES = 64 * QT / KW;
  constexpr int CPR = D / 8, N = 64 * CPR / 256;   // 16-byte chunks a row, and of a thread
  constexpr size_t kTileBytes = sizeof(T) * 64 * ROW;
  constexpr size_t kBytes = 2 * kTileBytes + sizeof(float) * 4 * 16 * KT * 16;
  __shared__ __align__(16) char smem[kBytes > kJoinBytes<D> ? kBytes : kJoinBytes<D>];
  __shared__ int sh_odd[2];
  __shared__ __align__(16) float sh_scales[2][CODE != 0 ? 64 : 4];   // of keys and values
  const PagedRel& r = a.rel;
  const unsigned all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;
  const unsigned groups = (rows + QUERIES - 1) / QUERIES;
  const unsigned of8 = blockIdx.x / 8u, item = of8 / groups * 8u + blockIdx.x % 8u;
  const int row0 = static_cast<int>(of8 % groups) * QUERIES;
  const int head = static_cast<int>(item % all_heads);
  const int x = static_cast<int>(item / all_heads);
  const Piece p = find_piece<WIN>(a, x);
  if (p.seq < 0) return;
  const int th = head / a.heads, kh = head % a.heads;
  if (a.meta && p.index == 0 && head == 0 && row0 == 0 && threadIdx.x == 0)
    a.meta[p.seq] = make_int2(x, p.count);

  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, lr = lane & 15;
  const int wrow = row0 + wave / KW * 16 * QT;  // the wave's first query
  const int key0 = wave % KW * 16 * KT;        // and first key of a tile
  Query<T, D, WIN> q[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
    q[qt] = Query<T, D, WIN>(a, p, th, kh, wrow + 16 * qt + lr, rows, g);
  // What the wave's oldest and newest queries see, and the workgroup's.
  auto sees = [&](int row) {
    return Sight<WIN>(a, p.length - (r.queries - 1 - min(row, rows - 1) / a.group));
  };
  const Sight<WIN> oldest = sees(wrow), newest = sees(wrow + 16 * QT - 1);
  const Sight<WIN> all_oldest = sees(row0), all_newest = sees(row0 + QUERIES - 1);
  const int high = WIN ? all_newest.limit : min(all_newest.limit, p.tile1 * kTile);
  const CT* kb = static_cast<const CT*>(a.k) + th * a.ks_table + kh * a.ks_head;
  const CT* vb = static_cast<const CT*>(a.v) + th * a.vs_table + kh * a.vs_head;
  const int32_t* table = r.table + p.seq * r.seq_stride + th * r.head_stride;
  T* ks = reinterpret_cast<T*>(smem);
  VT* vs = reinterpret_cast<VT*>(smem + kTileBytes);
  float* weights = reinterpret_cast<float*>(smem + 2 * kTileBytes) + wave * 16 * KT * 16;

  auto start = [&](int tile) { return (WIN ? p.at(tile, 1) : tile) * kTile; };
  auto page_id = [&](int tile) {
    const int pos = min(start(tile) + lane, r.pages_per_seq * r.page_size - 1);
    return table[static_cast<unsigned>(pos) / static_cast<unsigned>(r.page_size)];
  };
  auto slot_of = [&](int tile, int id) {
    const unsigned pos = start(tile) + lane;
    const bool there = static_cast<int>(pos) < high &&
                       (!WIN || static_cast<int>(pos) >= all_oldest.from ||
                        static_cast<int>(pos) < all_oldest.sinks) &&
                       static_cast<unsigned>(id) < static_cast<unsigned>(r.num_pages);
    return there ? id * r.page_size + static_cast<int>(pos % static_cast<unsigned>(r.page_size))
                 : -1;
  };
  // Chunk threadIdx.x + 256 i of a tile is row / CPR, column % CPR.
  Raw kr[N], vr[N];
  float kscale = 0.f, vscale = 0.f;   // CODE: of key `lane`, in every wave
  auto load = [&](int slot) {
    if constexpr (CODE != 0) {
      const unsigned block = static_cast<unsigned>(max(slot, 0)) / a.block;
      const int64_t at = static_cast<int64_t>(block) * all_heads + head;
      kscale = slot < 0 ? 0.f : a.k_scales[at];
      vscale = slot < 0 ? 0.f : a.v_scales[at];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + 256 * i;
      const int s = __shfl(slot, at / CPR, 64);
      kr[i] = *reinterpret_cast<const Raw*>(kb + max(s, 0) * a.ks_slot + at % CPR * 8);
      vr[i] = *reinterpret_cast<const Raw*>(vb + max(s, 0) * a.vs_slot + at % CPR * 8);
      if (s < 0) vr[i] = Raw{};   // a key that is not there
    }
  };

  float m[QT], l[QT];
  f32x4 o[QT][D / 16];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m[qt] = kNegInf;
    l[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Tiles of this workgroup: those of the piece that one of its queries may see (a
  // window's oldest queries are the sequence's, not this workgroup's).
  int first = p.tile0, last = (high + kTile - 1) / kTile;
  if constexpr (WIN) {
    last = min(p.tile1, last - (last > p.gap.sinks ? p.gap.skip : 0));
    if (first >= p.gap.sinks)
      first = max(first, max(all_oldest.from, 0) / kTile - p.gap.skip);
  }
  if (threadIdx.x < 2) sh_odd[threadIdx.x] = 0;
  int slot = -1, next_id = 0;
  if (first < last) {
    slot = slot_of(first, page_id(first));
    load(slot);
    next_id = page_id(first + 1);
  }
  for (int tile = first; tile < last; ++tile) {
    __syncthreads();   // the tile before has been read
    Largest<VT> largest;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + 256 * i;
      vec8<T> kk;
      vec8<VT> vv;
      if constexpr (CODE == 0) {
        kk = kr[i];
        vv = vr[i];
      } else {
        kk = __builtin_bit_cast(vec8<T>, code_octet<T, CODE>(kr[i]));
        vv = __builtin_bit_cast(vec8<VT>, code_octet<VT, CODE>(vr[i]));
      }
      if (CODE != TGX_CODE_INT8) largest.see(vv);
      *reinterpret_cast<vec8<T>*>(ks + at / CPR * ROW + at % CPR * 8) = kk;
      *reinterpret_cast<vec8<VT>*>(vs + at / CPR * ROW + at % CPR * 8) = vv;
    }
    bool strange = largest.odd();
    if constexpr (CODE != 0) {
      if (wave == 0) {
        sh_scales[0][lane] = kscale * a.scale_log2;
        sh_scales[1][lane] = vscale;
      }
      strange |= !(fabsf(vscale) < __builtin_huge_valf());
    }
    if (strange) sh_odd[tile & 1] = 1;
    if (threadIdx.x == 0) sh_odd[(tile + 1) & 1] = 0;
    __syncthreads();
    const unsigned long long gone = __ballot(slot < 0);
    if (tile + 1 < last) {
      slot = slot_of(tile + 1, next_id);
      next_id = page_id(tile + 2);
      load(slot);
    }
    const int pos = start(tile) + key0;
    if (wrow >= rows || pos >= newest.limit) continue;
    f32x4 c[QT][KT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) c[qt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const vec8<T> kf = *reinterpret_cast<const vec8<T>*>(
            ks + (key0 + 16 * kt + lr) * ROW + 32 * kc + 8 * g);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) c[qt][kt] = mfma(kf, q[qt].f[kc], c[qt][kt]);
      }
    f32x4 by[KT];   // CODE: the values' scales
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      if constexpr (CODE != 0) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(&sh_scales[0][key0 + 16 * kt + 4 * g]);
        by[kt] = *reinterpret_cast<const f32x4*>(&sh_scales[1][key0 + 16 * kt + 4 * g]);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) c[qt][kt] *= s;
      }
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if constexpr (CODE == 0) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) c[qt][kt] *= a.scale_log2;
      }
      weigh<VT, WIN>(c[qt], gone || !oldest.all(pos, 16 * KT, newest), gone >> key0, pos,
                     q[qt].sees, g, m[qt], l[qt], o[qt]);
      if constexpr (CODE != 0) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) c[qt][kt] *= by[kt];
      }
    }
    // (What does not fit the registers is then kept in memory beside the rare case only:
    // 512 new tokens 297 -> 285 us.)
    if (__builtin_expect(!sh_odd[tile & 1], 1)) {
      add_values<VT, D, KT, QT>(vs + key0 * ROW, c, g, lr, o);
    } else {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        add_seen_values<VT, D, WIN>(vs + key0 * ROW, c[qt], g, lr, pos, q[qt].sees, weights, o[qt]);
    }
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
    join_waves<T, D, KW>(a, p, x, head, th, kh, row0 + 16 * qt, 16 * QT, rows, smem, m[qt], l[qt],
                         o[qt]);
}

// Joins the pieces of each (sequence, head, query), a workgroup per query: each
// of its 256 / LPK lane groups takes every 256 / LPK-th piece, the next one's
// loads in flight; groups and waves are then merged in a fixed order.
template <int DT, int LPK>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  const PagedRel& r = a.rel;
  const int all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;
  const unsigned item = blockIdx.x / static_cast<unsigned>(rows);
  const int row = static_cast<int>(blockIdx.x % static_cast<unsigned>(rows));
  const int head = static_cast<int>(item % static_cast<unsigned>(all_heads));
  const int b = static_cast<int>(item / static_cast<unsigned>(all_heads));
  const int2 m = a.meta[b];
  if (m.y <= 1) return;
  const int wave = threadIdx.x >> 6, lane = lane_id(), part = lane % LPK, sub = lane / LPK;
  const bool has = 8 * part < a.D;
  State8 s;
  s.init();
  const int64_t stride = static_cast<int64_t>(all_heads) * rows * (a.D + 2);
  const float* src = a.partial + (static_cast<int64_t>(m.x) * all_heads + head) * rows * (a.D + 2) +
                     static_cast<int64_t>(row) * (a.D + 2);
  float o[8], om = kNegInf, ol = 0.f;
  auto load = [&](int j) {
    const bool there = j < m.y;
    const float* p = src + (there ? j : 0) * stride;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = has ? p[8 * part + i] : 0.f;
    om = there ? p[a.D] : kNegInf;
    ol = p[a.D + 1];
  };
  const int first = wave * (64 / LPK) + sub;
  load(first);
  for (int j = first; j < m.y; j += 256 / LPK) {
    float c[8], cm = om, cl = ol;
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = o[i];
    load(j + 256 / LPK);
    s.merge(cm, cl, c);
  }
#pragma unroll
  for (int mask = LPK; mask < 64; mask <<= 1) s.merge_xor(mask);
  __shared__ float ml[4][2];
  __shared__ float acc[4][8 * LPK];
  if (sub == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[wave][8 * part + i] = s.acc[i];
    if (part == 0) {
      ml[wave][0] = s.m;
      ml[wave][1] = s.l;
    }
  }
  __syncthreads();
  if (wave != 0 || sub != 0 || !has) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = acc[w][8 * part + i];
    s.merge(ml[w][0], ml[w][1], c);
  }
  const int th = head / a.heads, kh = head % a.heads;
  const int t = row / a.group, g = row % a.group;
  const int64_t q_row = (static_cast<int64_t>(b) * r.queries + t) * r.heads + th;
  const float inv = s.l == 0.f ? 0.f : 1.f / s.l;
#pragma unroll
  for (int i = 0; i < 8; ++i) s.acc[i] *= inv;
  V::store(static_cast<T*>(a.out) + ((q_row * a.heads + kh) * a.group + g) * a.D + 8 * part,
           s.acc);
}


}  // namespace
}  // namespace tgx
