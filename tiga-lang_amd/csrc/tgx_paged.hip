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
// Bound: a cached row has to be read once, 4 * D bytes a key and head at 16
// bits, against 4 * group * D operations a new token: memory, for any group a
// model has and few new tokens.  The matrix tiles (16 bits, D = 32, 64, 128) read it
// once for 128 queries of its key head; paged_rows_kernel, which takes every other
// width and fp32, once for each query.
//
// Work split.  Lengths are only known on the device, so the launch is sized
// from the host's bounds and every workgroup finds its piece itself: the keys
// of all sequences, in tiles of 64, are cut into pieces of at most `c` tiles,
// c at least kMinTiles and just large enough for W pieces to cover them all;
// sequence b gets k_b = max(1, ceil(tiles_b / c)) pieces of equal size, W
// together where there are fewer than W / 2 sequences, W + n_seqs at most.  A
// sequence of one piece writes its output; of several, each piece writes its
// running maximum, sum and unnormalized output, which a second launch joins in
// piece order.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "tgx_device.h"
#include "tgx_host.h"
#include "tgx_paged.h"
#include "tgx_profile.h"
#include "tgx_vals.h"

namespace tgx {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;       // keys a tile
constexpr int kMinTiles = 4;    // tiles a piece has at least, where the sequence has them

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
};

// 2^x on the hardware unit: exact 0 for -inf.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

struct Piece {
  int seq;        // -1: no such piece
  int length;     // cached tokens of the sequence
  int index;      // piece of the sequence
  int count;      // pieces of the sequence
  int tile0, tile1;
};

// Cuts n tiles into p.count pieces whose sizes differ by one at most.
__device__ __forceinline__ void cut_tiles(Piece& p, int n) {
  const int each = n / p.count, more = n % p.count;
  p.tile0 = p.index * each + min(p.index, more);
  p.tile1 = p.tile0 + each + (p.index < more);
}

// Piece `x` of the launch; every wave finds it by itself.  Lane l looks
// after the sequences [l, l + 1) * ceil(n / 64).
__device__ __forceinline__ Piece find_piece(const PagedRel& r, int pieces, bool whole, int x) {
  Piece p{-1, 0, 0, 1, 0, 0};
  if (whole) {   // one piece a sequence
    if (x >= r.n_seqs) return p;
    p.seq = x;
    p.length = paged_length(r, x);
    p.tile1 = (p.length + kTile - 1) / kTile;
    return p;
  }
  const int lane = lane_id();
  if (r.n_seqs == 1) {
    p.length = paged_length(r, 0);
    const int n = (p.length + kTile - 1) / kTile;
    const int c = max(kMinTiles, (n + pieces - 1) / pieces);
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
  for (int b = b0; b < b1; ++b) tiles += (paged_length(r, b) + kTile - 1) / kTile;
  const int total = read_lane(wave_prefix(tiles), 63);
  // Rounding up adds a piece a sequence at most, which are taken off first.
  const int room = max(pieces - r.n_seqs, (pieces + 1) / 2);
  const int c = max(kMinTiles, (total + room - 1) / room);
  int mine = 0;
  if (per == 1)
    mine = b0 < b1 ? max(1, (tiles + c - 1) / c) : 0;
  else
    for (int b = b0; b < b1; ++b)
      mine += max(1, ((paged_length(r, b) + kTile - 1) / kTile + c - 1) / c);
  const int end = wave_prefix(mine);
  const unsigned long long hit = __ballot(x < end && x >= end - mine);
  if (!hit) return p;
  const int owner = __builtin_ctzll(hit);
  int at = end - mine, found = -1, k = 1, n = 0, len = 0;
  for (int b = b0; b < b1 && found < 0; ++b) {
    len = paged_length(r, b);
    n = (len + kTile - 1) / kTile;
    k = max(1, (n + c - 1) / c);
    if (x < at + k) found = b;
    else at += k;
  }
  p.seq = read_lane(found, owner);
  p.length = read_lane(len, owner);
  p.count = read_lane(k, owner);
  p.index = x - read_lane(at, owner);
  cut_tiles(p, read_lane(n, owner));
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
template <int DT, int LPK>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  const PagedRel& r = a.rel;
  const int all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;   // queries of one (sequence, head)
  const unsigned item = blockIdx.x / static_cast<unsigned>(rows);
  const int row = static_cast<int>(blockIdx.x % static_cast<unsigned>(rows));
  const int head = static_cast<int>(item % static_cast<unsigned>(all_heads));
  const int x = static_cast<int>(item / static_cast<unsigned>(all_heads));
  const Piece p = find_piece(r, a.pieces, a.meta == nullptr, x);
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
  const T* kb = static_cast<const T*>(a.k) + th * a.ks_table + kh * a.ks_head + 8 * part;
  const T* vb = static_cast<const T*>(a.v) + th * a.vs_table + kh * a.vs_head + 8 * part;
  const int32_t* table = r.table + p.seq * r.seq_stride + th * r.head_stride;

  const int limit = min(p.length - (r.queries - 1 - t), p.tile1 * kTile);
  State8 s;
  s.init();
  for (int j = p.tile0 * kTile + wave * (64 / LPK) + sub; j < limit; j += 4 * (64 / LPK)) {
    const int slot = paged_slot(r, table, j);
    if (slot < 0) continue;
    float kv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float vv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (has) {
      const typename V::Raw kr = V::load(kb + slot * a.ks_slot);
      const typename V::Raw vr = V::load(vb + slot * a.vs_slot);
      V::unpack(kr, kv);
      V::unpack(vr, vv);
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) dot += q[i] * kv[i];
    s.merge(group_sum<LPK>(dot) * a.scale_log2, 1.f, vv);
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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
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
template <typename T, int D>
struct Query {
  vec8<T> f[D / 32];
  int limit;
  Query() = default;
  __device__ __forceinline__ Query(const PagedArgs& a, const Piece& p, int th, int kh, int row,
                                   int rows, int g) {
    const int t = min(row / a.group, a.rel.queries - 1), gq = row % a.group;
    limit = p.length - (a.rel.queries - 1 - t);
    const int64_t q_row = (static_cast<int64_t>(p.seq) * a.rel.queries + t) * a.rel.heads + th;
    const T* q = static_cast<const T*>(a.q) + q_row * a.qs_row + kh * a.qs_head +
                 gq * a.qs_group + 8 * g;
#pragma unroll
    for (int kc = 0; kc < D / 32; ++kc)
      f[kc] = row < rows ? *reinterpret_cast<const vec8<T>*>(q + 32 * kc) : vec8<T>{};
  }
};

// Scores of 16 KT keys from position `pos` become weights 2^(s - m + lift) under
// the running maximum m; l and o follow it.  `gone`: bit k set, key k is not
// there; `masked`: some key may be hidden from the lane's query.
template <typename T, int KT, int DT>
__device__ __forceinline__ void weigh(f32x4 (&c)[KT], float scale, bool masked,
                                      unsigned long long gone, int pos, int limit, int g,
                                      float& m, float& l, f32x4 (&o)[DT]) {
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) c[kt] *= scale;
  if (masked) {
    gone >>= 4 * g;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((gone >> (16 * kt + i) & 1) || pos + 16 * kt + 4 * g + i >= limit) c[kt][i] = kNegInf;
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
template <typename T, int D, int KT>
__device__ __forceinline__ void add_seen_values(const T* v, const f32x4 (&c)[KT], int g, int lr,
                                                int pos, int limit, float* weights,
                                                f32x4 (&o)[D / 16]) {
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) weights[(16 * kt + 4 * g + i) * 16 + lr] = c[kt][i];
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  for (int key = 0; key < 16 * KT; ++key) {
    if (pos + key >= limit) continue;
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
template <typename T, int D>
__global__ __launch_bounds__(256, (D == 128 ? 2 : D == 64 ? 3 : 4)) void paged_tile_kernel(
    PagedArgs a) {
  constexpr int KT = KEYS / 16, KC = D / 32, ROW = kRow<D>;
  constexpr size_t kStage = sizeof(T) * 4 * KEYS * ROW;
  constexpr size_t kBytes = kStage + sizeof(float) * 4 * KEYS * 16;
  __shared__ __align__(16) char smem[kBytes > kJoinBytes<D> ? kBytes : kJoinBytes<D>];
  const PagedRel& r = a.rel;
  const unsigned all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;
  const int head = static_cast<int>(blockIdx.x % all_heads);
  const int x = static_cast<int>(blockIdx.x / all_heads);
  const Piece p = find_piece(r, a.pieces, a.meta == nullptr, x);
  if (p.seq < 0) return;
  const int th = head / a.heads, kh = head % a.heads;
  if (a.meta && p.index == 0 && head == 0 && threadIdx.x == 0)
    a.meta[p.seq] = make_int2(x, p.count);

  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, lr = lane & 15;
  const Query<T, D> q(a, p, th, kh, lr, rows, g);
  // The fewest and most positions any of the queries sees.
  const int low = p.length - (r.queries - 1);
  const int high = min(p.length, p.tile1 * kTile);
  const T* kb = static_cast<const T*>(a.k) + th * a.ks_table + kh * a.ks_head + 8 * g;
  const T* vb = static_cast<const T*>(a.v) + th * a.vs_table + kh * a.vs_head + 8 * g;
  const int32_t* table = r.table + p.seq * r.seq_stride + th * r.head_stride;
  // The wave's staged V, and its weights where they are taken key by key.
  T* stage = reinterpret_cast<T*>(smem) + wave * KEYS * ROW;
  float* weights = reinterpret_cast<float*>(smem + kStage) + wave * KEYS * 16;

  // Steps of this wave: first + 4 i < last.  Lane l keeps the page id of key
  // l (mod KEYS) of a step.
  const int first = p.tile0 * (kTile / KEYS) + wave;
  const int last = (high + KEYS - 1) / KEYS;
  auto page_id = [&](int step) {
    const int pos = min(step * KEYS + lane % KEYS, r.pages_per_seq * r.page_size - 1);
    return table[static_cast<unsigned>(pos) / static_cast<unsigned>(r.page_size)];
  };
  auto slot_of = [&](int step, int id) {
    const unsigned pos = step * KEYS + lane % KEYS;
    const bool there = static_cast<int>(pos) < high &&
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
    int next_id = page_id(first + 4);
    for (int step = first; step < last; step += 4) {
      const int next = slot_of(step + 4, next_id);
      next_id = page_id(step + 8);
      const unsigned long long gone = __ballot(slot < 0);   // bit k: key k is not there
      f32x4 c[1][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) c[0][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kc = 0; kc < KC; ++kc)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) c[0][kt] = mfma(kf[kt][kc], q.f[kc], c[0][kt]);
      load(kf, kb, a.ks_slot, next);

      const bool tail = step * KEYS + KEYS > low;   // some query sees only a part
      weigh<T>(c[0], a.scale_log2, gone || tail, gone, step * KEYS, q.limit, g, m, l, o[0]);

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
        add_seen_values<T, D, KT>(stage, c[0], g, lr, step * KEYS, q.limit, weights, o[0]);
      slot = next;
    }
  }
  join_waves<T, D, 4>(a, p, x, head, th, kh, 0, 16, rows, smem, m, l, o[0]);
}

// More than 16 queries.  The four waves stage 64 keys together, the next tile's
// loads in flight in registers while this one is multiplied.  KW waves share
// 16 QT queries and take 64 / KW keys of a tile each, so a workgroup holds 64 QT
// / KW queries: 32 (KW = 2), 64, or 128 (QT = 2), the smallest that holds all
// of them (one read of the keys), 128 where none does.  Workgroups of the same
// keys are 8 apart, on one XCD's L2.
template <typename T, int D, int KW, int QT>
__global__ __launch_bounds__(256, (D == 128 || QT == 2 ? 2 : 3)) void paged_block_kernel(
    PagedArgs a) {
  constexpr int KT = 4 / KW, KC = D / 32, ROW = kRow<D>, QUERIES = 64 * QT / KW;
  constexpr int CPR = D / 8, N = 64 * CPR / 256;   // 16-byte chunks a row, and of a thread
  constexpr size_t kTileBytes = sizeof(T) * 64 * ROW;
  constexpr size_t kBytes = 2 * kTileBytes + sizeof(float) * 4 * 16 * KT * 16;
  __shared__ __align__(16) char smem[kBytes > kJoinBytes<D> ? kBytes : kJoinBytes<D>];
  __shared__ int sh_odd[2];
  const PagedRel& r = a.rel;
  const unsigned all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;
  const unsigned groups = (rows + QUERIES - 1) / QUERIES;
  const unsigned of8 = blockIdx.x / 8u, item = of8 / groups * 8u + blockIdx.x % 8u;
  const int row0 = static_cast<int>(of8 % groups) * QUERIES;
  const int head = static_cast<int>(item % all_heads);
  const int x = static_cast<int>(item / all_heads);
  const Piece p = find_piece(r, a.pieces, a.meta == nullptr, x);
  if (p.seq < 0) return;
  const int th = head / a.heads, kh = head % a.heads;
  if (a.meta && p.index == 0 && head == 0 && row0 == 0 && threadIdx.x == 0)
    a.meta[p.seq] = make_int2(x, p.count);

  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, lr = lane & 15;
  const int wrow = row0 + wave / KW * 16 * QT;  // the wave's first query
  const int key0 = wave % KW * 16 * KT;        // and first key of a tile
  Query<T, D> q[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
    q[qt] = Query<T, D>(a, p, th, kh, wrow + 16 * qt + lr, rows, g);
  // The fewest and most positions any of the wave's queries sees, and the most of the
  // workgroup's.
  auto sees = [&](int row) {
    return p.length - (r.queries - 1 - min(row, rows - 1) / a.group);
  };
  const int low = sees(wrow), wave_high = sees(wrow + 16 * QT - 1);
  const int high = min(sees(row0 + QUERIES - 1), p.tile1 * kTile);
  const T* kb = static_cast<const T*>(a.k) + th * a.ks_table + kh * a.ks_head;
  const T* vb = static_cast<const T*>(a.v) + th * a.vs_table + kh * a.vs_head;
  const int32_t* table = r.table + p.seq * r.seq_stride + th * r.head_stride;
  T* ks = reinterpret_cast<T*>(smem);
  T* vs = reinterpret_cast<T*>(smem + kTileBytes);
  float* weights = reinterpret_cast<float*>(smem + 2 * kTileBytes) + wave * 16 * KT * 16;

  auto page_id = [&](int tile) {
    const int pos = min(tile * kTile + lane, r.pages_per_seq * r.page_size - 1);
    return table[static_cast<unsigned>(pos) / static_cast<unsigned>(r.page_size)];
  };
  auto slot_of = [&](int tile, int id) {
    const unsigned pos = tile * kTile + lane;
    const bool there = static_cast<int>(pos) < high &&
                       static_cast<unsigned>(id) < static_cast<unsigned>(r.num_pages);
    return there ? id * r.page_size + static_cast<int>(pos % static_cast<unsigned>(r.page_size))
                 : -1;
  };
  // Chunk threadIdx.x + 256 i of a tile is row / CPR, column % CPR.
  vec8<T> kr[N], vr[N];
  auto load = [&](int slot) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + 256 * i;
      const int s = __shfl(slot, at / CPR, 64);
      kr[i] = *reinterpret_cast<const vec8<T>*>(kb + max(s, 0) * a.ks_slot + at % CPR * 8);
      vr[i] = *reinterpret_cast<const vec8<T>*>(vb + max(s, 0) * a.vs_slot + at % CPR * 8);
      if (s < 0) vr[i] = vec8<T>{};   // a key that is not there
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
  const int last = (high + kTile - 1) / kTile;
  if (threadIdx.x < 2) sh_odd[threadIdx.x] = 0;
  int slot = -1, next_id = 0;
  if (p.tile0 < last) {
    slot = slot_of(p.tile0, page_id(p.tile0));
    load(slot);
    next_id = page_id(p.tile0 + 1);
  }
  for (int tile = p.tile0; tile < last; ++tile) {
    __syncthreads();   // the tile before has been read
    Largest<T> largest;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + 256 * i;
      largest.see(vr[i]);
      *reinterpret_cast<vec8<T>*>(ks + at / CPR * ROW + at % CPR * 8) = kr[i];
      *reinterpret_cast<vec8<T>*>(vs + at / CPR * ROW + at % CPR * 8) = vr[i];
    }
    if (largest.odd()) sh_odd[tile & 1] = 1;
    if (threadIdx.x == 0) sh_odd[(tile + 1) & 1] = 0;
    __syncthreads();
    const unsigned long long gone = __ballot(slot < 0);
    if (tile + 1 < last) {
      slot = slot_of(tile + 1, next_id);
      next_id = page_id(tile + 2);
      load(slot);
    }
    const int pos = tile * kTile + key0;
    if (wrow >= rows || pos >= wave_high) continue;
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
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
      weigh<T>(c[qt], a.scale_log2, gone || pos + 16 * KT > low, gone >> key0, pos, q[qt].limit, g,
            m[qt], l[qt], o[qt]);
    if (!sh_odd[tile & 1]) {
      add_values<T, D, KT, QT>(vs + key0 * ROW, c, g, lr, o);
    } else {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        add_seen_values<T, D, KT>(vs + key0 * ROW, c[qt], g, lr, pos, q[qt].limit, weights, o[qt]);
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

// Whether the matrix tiles take the shape; the rows kernel takes every other.
bool tiled(int D, int dtype) {
  return dtype != TGX_DTYPE_F32 && (D == 32 || D == 64 || D == 128);
}

// Queries a workgroup holds.
int held_queries(const tgx_paged& p, int group, int D, int dtype) {
  if (!tiled(D, dtype)) return 1;
  const int64_t queries = static_cast<int64_t>(p.queries) * group;
  return queries <= 16 ? 16 : queries <= 32 ? 32 : queries <= 64 ? 64 : 128;
}

// Workgroups that read the same keys or another head's: those of one piece.
int64_t workgroups_per_piece(const tgx_paged& p, int heads, int group, int D, int dtype) {
  return static_cast<int64_t>(p.table_heads) * heads *
         ceil_div(static_cast<int64_t>(p.queries) * group, held_queries(p, group, D, dtype));
}

// How a launch is cut: W pieces wanted, pieces launched at most, and whether
// any sequence can have several.
struct Cut {
  int64_t wanted, launched;
  bool split;
};

// Workgroups wanted in all: four a CU.  The tile kernel holds two at once at D =
// 128, three at D = 64 and four at D = 32 (its launch bounds), so these are two
// full rounds, one and a third, and one.  Four sequences of 100k to 131k tokens, D =
// 128: 346 us with two rounds that fit, 368-420 us with rounds that end half full;
// more and smaller pieces pay for their first loads, fewer end unevenly.  (Ragged
// sequences do not fill the rounds: find_piece takes a piece a sequence off before
// it sizes them, 95 of 128 for 64 sequences of 100 to 4000.)  A workgroup of more
// than 64 queries writes and joins as much as it reads of a few tiles of keys:
// half as many (512 new tokens of four sequences: 315 us with four a CU, 282 us).
//
// Nothing is split where it cannot be (a table of kMinTiles), where one
// piece has as many workgroups as are wanted, where the join, a workgroup a
// query, would be more than one launch, and where short tables (up
// to kWholeTiles) of many sequences give every CU a workgroup: the join's
// launch costs more than the unevenness (32 sequences of 8 heads over 24
// pages of 64: attention 44 us, 36 us).
constexpr int kWholeTiles = 32;

Cut cut_of(const tgx_paged& p, int heads, int group, int D, int dtype) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  const int64_t each = workgroups_per_piece(p, heads, group, D, dtype);
  const int64_t tiles = ceil_div(static_cast<int64_t>(p.pages_per_seq) * p.page_size, kTile);
  const int64_t wanted = cus * (held_queries(p, group, D, dtype) > 64 ? 2 : 4) / each;
  const int64_t queries = static_cast<int64_t>(p.table_heads) * heads * p.queries * group;
  if (tiles <= kMinTiles || wanted <= 1 || p.n_seqs > kMaxBlocks256 / queries ||
      (tiles <= kWholeTiles && p.n_seqs * each >= cus))
    return Cut{1, p.n_seqs, false};
  return Cut{wanted, std::min(wanted + p.n_seqs, p.n_seqs * ceil_div(tiles, kMinTiles)), true};
}

int check_attn(const tgx_paged* p, int heads, int group, int D, int dtype) {
  if (int st = check_paged(p)) return st;
  TGX_REQUIRE(heads >= 1 && group >= 1, "heads and group must be positive");
  TGX_REQUIRE(dtype_bytes(dtype) != 0, "unknown dtype %d", dtype);
  if (D < 8 || D > 512 || D % 8) {
    set_error("head width %d: the paged attention takes multiples of 8 up to 512", D);
    return TGX_UNSUPPORTED;
  }
  const int64_t tiles = ceil_div(static_cast<int64_t>(p->pages_per_seq) * p->page_size, kTile);
  const int64_t rows = static_cast<int64_t>(group) * p->queries;
  TGX_REQUIRE(rows < (int64_t{1} << 28) && static_cast<int64_t>(p->table_heads) * heads < 1 << 28 &&
                  p->n_seqs * std::max<int64_t>(tiles, 1) < (int64_t{1} << 31),
              "paged attention: sizes past 32 bits");
  const int64_t each = workgroups_per_piece(*p, heads, group, D, dtype);
  if (each > kMaxBlocks256 ||
      cut_of(*p, heads, group, D, dtype).launched > kMaxBlocks256 / each - 8) {
    set_error("paged attention: too many sequences, heads and queries for one launch");
    return TGX_UNSUPPORTED;
  }
  return TGX_OK;
}

size_t meta_bytes(const tgx_paged& p) { return align_up(sizeof(int2) * p.n_seqs); }

template <int DT, int LPK>
int launch_rows(const PagedArgs& a, const Cut& cut, hipStream_t stream) {
  const int64_t queries = static_cast<int64_t>(a.rel.heads) * a.heads * a.rel.queries * a.group;
  TGX_PROFILE("paged_rows", stream);
  paged_rows_kernel<DT, LPK><<<dim3(static_cast<uint32_t>(cut.launched * queries)), dim3(256), 0,
                               stream>>>(a);
  TGX_LAUNCHED("paged_rows");
  return TGX_OK;
}

template <int DT, int LPK>
int launch_join(const PagedArgs& a, hipStream_t stream) {
  const int64_t queries = static_cast<int64_t>(a.rel.heads) * a.heads * a.rel.queries * a.group;
  TGX_PROFILE("paged_join", stream);
  paged_join_kernel<DT, LPK>
      <<<dim3(static_cast<uint32_t>(a.rel.n_seqs * queries)), dim3(256), 0, stream>>>(a);
  TGX_LAUNCHED("paged_join");
  return TGX_OK;
}

template <int DT>
int dispatch_rows(const PagedArgs& a, const Cut& cut, hipStream_t stream) {
  if (a.D <= 32) return launch_rows<DT, 4>(a, cut, stream);
  if (a.D <= 64) return launch_rows<DT, 8>(a, cut, stream);
  if (a.D <= 128) return launch_rows<DT, 16>(a, cut, stream);
  if (a.D <= 256) return launch_rows<DT, 32>(a, cut, stream);
  return launch_rows<DT, 64>(a, cut, stream);
}

template <int DT>
int dispatch_join(const PagedArgs& a, hipStream_t stream) {
  if (a.D <= 32) return launch_join<DT, 4>(a, stream);
  if (a.D <= 64) return launch_join<DT, 8>(a, stream);
  if (a.D <= 128) return launch_join<DT, 16>(a, stream);
  if (a.D <= 256) return launch_join<DT, 32>(a, stream);
  return launch_join<DT, 64>(a, stream);
}

template <typename T, int D>
int launch_tiles(const PagedArgs& a, const Cut& cut, int held, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.rel.queries) * a.group;
  const int64_t pieces = cut.launched * a.rel.heads * a.heads;
  TGX_PROFILE("paged_tiles", stream);
  if (held == 16) {
    paged_tile_kernel<T, D><<<dim3(static_cast<uint32_t>(pieces)), dim3(256), 0, stream>>>(a);
  } else {
    const dim3 grid(static_cast<uint32_t>(ceil_div(pieces, 8) * 8 * ceil_div(rows, held)));
    if (held == 32) paged_block_kernel<T, D, 2, 1><<<grid, dim3(256), 0, stream>>>(a);
    else if (held == 64) paged_block_kernel<T, D, 1, 1><<<grid, dim3(256), 0, stream>>>(a);
    else paged_block_kernel<T, D, 1, 2><<<grid, dim3(256), 0, stream>>>(a);
  }
  TGX_LAUNCHED("paged_tiles");
  return TGX_OK;
}

template <typename T>
int dispatch_tiles(const PagedArgs& a, const Cut& cut, int held, hipStream_t stream) {
  if (a.D == 32) return launch_tiles<T, 32>(a, cut, held, stream);
  if (a.D == 64) return launch_tiles<T, 64>(a, cut, held, stream);
  return launch_tiles<T, 128>(a, cut, held, stream);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_paged_attn_workspace(const tgx_paged* p, int heads, int group, int D,
                                        int dtype, size_t* bytes) {
  TGX_REQUIRE(bytes != nullptr, "null bytes");
  if (int st = check_attn(p, heads, group, D, dtype)) return st;
  const int64_t groups = static_cast<int64_t>(p->table_heads) * heads;
  const Cut cut = cut_of(*p, heads, group, D, dtype);
  *bytes = !cut.split ? 0
                      : meta_bytes(*p) + sizeof(float) * cut.launched * groups * group *
                                             p->queries * (D + 2);
  return TGX_OK;
}

extern "C" int tgx_paged_attn(const tgx_paged* p, const void* q_dev, const void* k_dev,
                              const void* v_dev, const int64_t* strides, float scale,
                              void* out_dev, int heads, int group, int D, int dtype,
                              void* workspace_dev, size_t workspace_bytes, void* stream) {
  if (int st = check_attn(p, heads, group, D, dtype)) return st;
  if (p->n_seqs == 0) return TGX_OK;
  TGX_REQUIRE(q_dev && out_dev && strides, "null operand");
  TGX_REQUIRE(p->num_pages == 0 || (k_dev && v_dev), "null cache");
  TGX_REQUIRE(aligned16(q_dev) && aligned16(k_dev) && aligned16(v_dev) && aligned16(out_dev),
              "q, k, v and out must start on 16 bytes");
  const int vec = 16 / dtype_bytes(dtype);
  for (int i = 0; i < 9; ++i)
    TGX_REQUIRE(strides[i] % vec == 0, "stride %lld does not keep rows on 16 bytes",
                static_cast<long long>(strides[i]));
  size_t need = 0;
  if (int st = tgx_paged_attn_workspace(p, heads, group, D, dtype, &need)) return st;
  TGX_REQUIRE(workspace_bytes >= need && (need == 0 || workspace_dev),
              "workspace of %zu bytes, needs %zu", workspace_bytes, need);
  const Cut cut = cut_of(*p, heads, group, D, dtype);
  PagedArgs a{};
  a.rel = paged_rel(*p);
  // Without pages there is no slot to read, whatever the lengths say.
  if (p->num_pages == 0) a.rel.pages_per_seq = 0;
  a.q = q_dev;
  a.k = k_dev;
  a.v = v_dev;
  a.qs_row = strides[0], a.qs_head = strides[1], a.qs_group = strides[2];
  a.ks_slot = strides[3], a.ks_table = strides[4], a.ks_head = strides[5];
  a.vs_slot = strides[6], a.vs_table = strides[7], a.vs_head = strides[8];
  a.out = out_dev;
  a.scale_log2 = scale * kLog2e;
  a.heads = heads;
  a.group = group;
  a.D = D;
  a.pieces = static_cast<int>(cut.wanted);
  if (cut.split) {
    a.meta = static_cast<int2*>(workspace_dev);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace_dev) + meta_bytes(*p));
  }
  hipStream_t s = as_stream(stream);
  const bool tiles = tiled(D, dtype);
  const int held = held_queries(*p, group, D, dtype);
  int st;
  switch (dtype) {
    case TGX_DTYPE_BF16:
      st = tiles ? dispatch_tiles<__bf16>(a, cut, held, s)
                 : dispatch_rows<TGX_DTYPE_BF16>(a, cut, s);
      return st || !cut.split ? st : dispatch_join<TGX_DTYPE_BF16>(a, s);
    case TGX_DTYPE_F16:
      st = tiles ? dispatch_tiles<_Float16>(a, cut, held, s)
                 : dispatch_rows<TGX_DTYPE_F16>(a, cut, s);
      return st || !cut.split ? st : dispatch_join<TGX_DTYPE_F16>(a, s);
    default:
      st = dispatch_rows<TGX_DTYPE_F32>(a, cut, s);
      return st || !cut.split ? st : dispatch_join<TGX_DTYPE_F32>(a, s);
  }
}
