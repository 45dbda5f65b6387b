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
// Bound: every cached row is read once, 4 * D bytes a key and head at 16
// bits, against 4 * group * D operations: memory, for any group a model has.
//
// Work split.  Lengths are only known on the device, so the launch is sized
// from the host's bounds and every workgroup finds its piece itself: the keys
// of all sequences, in tiles of 64, are cut into pieces of at most `c` tiles,
// c the smallest number (at least kMinTiles) for which W pieces cover them
// all; sequence b gets k_b = max(1, ceil(tiles_b / c)) pieces of equal size,
// at most W + n_seqs together.  A sequence of one piece writes its output; of
// several, each piece writes its running maximum, sum and unnormalized
// output, which a second launch joins in piece order.
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

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
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
  const int per = (r.n_seqs + 63) / 64;
  const int b0 = lane * per, b1 = min(r.n_seqs, b0 + per);
  int tiles = 0;
  for (int b = b0; b < b1; ++b) tiles += (paged_length(r, b) + kTile - 1) / kTile;
  const int total = wave_sum(tiles);
  const int c = max(kMinTiles, (total + pieces - 1) / pieces);
  int mine = 0;
  for (int b = b0; b < b1; ++b)
    mine += max(1, ((paged_length(r, b) + kTile - 1) / kTile + c - 1) / c);
  int end = mine;   // inclusive prefix over the lanes
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(end, d, 64);
    if (lane >= d) end += o;
  }
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
  n = read_lane(n, owner);
  p.tile0 = static_cast<int>(static_cast<int64_t>(p.index) * n / p.count);
  p.tile1 = static_cast<int>(static_cast<int64_t>(p.index + 1) * n / p.count);
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
// groups and the four waves are merged at the end.
template <int DT, int LPK>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  const PagedRel& r = a.rel;
  const int all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;   // queries of one (sequence, head)
  const int64_t item = blockIdx.x;
  const int row = static_cast<int>(item % rows);
  const int head = static_cast<int>(item / rows % all_heads);
  const int x = static_cast<int>(item / rows / all_heads);
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

// Joins the pieces of each (sequence, head, query) in a fixed order: a wave per query.
template <int DT, int LPK>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  const PagedRel& r = a.rel;
  const int all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= static_cast<int64_t>(r.n_seqs) * all_heads * rows) return;
  const int row = static_cast<int>(item % rows);
  const int head = static_cast<int>(item / rows % all_heads);
  const int b = static_cast<int>(item / rows / all_heads);
  const int2 m = a.meta[b];
  if (m.y <= 1) return;
  const int lane = lane_id(), part = lane % LPK, sub = lane / LPK;
  const bool has = 8 * part < a.D;
  State8 s;
  s.init();
  for (int j = sub; j < m.y; j += 64 / LPK) {
    const float* src = a.partial +
                       ((static_cast<int64_t>(m.x + j) * all_heads + head) * rows + row) *
                           (a.D + 2);
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = has ? src[8 * part + i] : 0.f;
    s.merge(src[a.D], src[a.D + 1], o);
  }
#pragma unroll
  for (int mask = LPK; mask < 64; mask <<= 1) s.merge_xor(mask);
  if (sub != 0 || !has) return;
  const int th = head / a.heads, kh = head % a.heads;
  const int t = row / a.group, g = row % a.group;
  const int64_t q_row = (static_cast<int64_t>(b) * r.queries + t) * r.heads + th;
  const float inv = s.l == 0.f ? 0.f : 1.f / s.l;
#pragma unroll
  for (int i = 0; i < 8; ++i) s.acc[i] *= inv;
  V::store(static_cast<T*>(a.out) + ((q_row * a.heads + kh) * a.group + g) * a.D + 8 * part,
           s.acc);
}

// How a launch is cut: W pieces wanted for each head's query group, pieces
// launched at most, and whether any sequence can have several.
struct Cut {
  int64_t wanted, launched;
  bool split;
};

// Workgroups wanted in all: what the GPU holds at once, several times over, so
// that pieces of uneven length even out.
int64_t wanted_workgroups() {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  return static_cast<int64_t>(cus) * 8;
}

Cut cut_of(const tgx_paged& p, int64_t groups) {
  const int64_t tiles = ceil_div(static_cast<int64_t>(p.pages_per_seq) * p.page_size, kTile);
  if (tiles <= kMinTiles) return Cut{1, p.n_seqs, false};
  const int64_t wanted = std::max<int64_t>(1, wanted_workgroups() / groups);
  const int64_t most = p.n_seqs * ceil_div(tiles, kMinTiles);
  return Cut{wanted, std::min(wanted + p.n_seqs, most), true};
}

int check_attn(const tgx_paged* p, int heads, int group, int D, int dtype) {
  if (int st = check_paged(p)) return st;
  TGX_REQUIRE(heads >= 1 && group >= 1, "heads and group must be positive");
  TGX_REQUIRE(dtype_bytes(dtype) != 0, "unknown dtype %d", dtype);
  if (D < 8 || D > 512 || D % 8) {
    set_error("head width %d: the paged attention takes multiples of 8 up to 512", D);
    return TGX_UNSUPPORTED;
  }
  const int64_t queries = static_cast<int64_t>(p->table_heads) * heads * group * p->queries;
  const int64_t tiles = ceil_div(static_cast<int64_t>(p->pages_per_seq) * p->page_size, kTile);
  TGX_REQUIRE(queries < (int64_t{1} << 28) &&
                  p->n_seqs * std::max<int64_t>(tiles, 1) < (int64_t{1} << 31) &&
                  (p->n_seqs + wanted_workgroups()) * queries <= kMaxBlocks256,
              "paged attention: too many sequences, heads and queries for one launch");
  return TGX_OK;
}

size_t meta_bytes(const tgx_paged& p) { return align_up(sizeof(int2) * p.n_seqs); }

template <int DT, int LPK>
int launch_rows(const PagedArgs& a, const Cut& cut, hipStream_t stream) {
  const int64_t queries = static_cast<int64_t>(a.rel.heads) * a.heads * a.rel.queries * a.group;
  {
    TGX_PROFILE("paged_rows", stream);
    paged_rows_kernel<DT, LPK><<<dim3(static_cast<uint32_t>(cut.launched * queries)), dim3(256),
                                 0, stream>>>(a);
  }
  TGX_LAUNCHED("paged_rows");
  if (!cut.split) return TGX_OK;
  {
    TGX_PROFILE("paged_join", stream);
    paged_join_kernel<DT, LPK>
        <<<dim3(static_cast<uint32_t>(ceil_div(a.rel.n_seqs * queries, 4))), dim3(256), 0,
           stream>>>(a);
  }
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

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_paged_attn_workspace(const tgx_paged* p, int heads, int group, int D,
                                        int dtype, size_t* bytes) {
  TGX_REQUIRE(bytes != nullptr, "null bytes");
  if (int st = check_attn(p, heads, group, D, dtype)) return st;
  const int64_t groups = static_cast<int64_t>(p->table_heads) * heads;
  const Cut cut = cut_of(*p, groups * group * p->queries);
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
  const Cut cut = cut_of(*p, static_cast<int64_t>(p->table_heads) * heads * group * p->queries);
  PagedArgs a{};
  a.rel = paged_rel(*p);
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
  switch (dtype) {
    case TGX_DTYPE_BF16: return dispatch_rows<TGX_DTYPE_BF16>(a, cut, as_stream(stream));
    case TGX_DTYPE_F16: return dispatch_rows<TGX_DTYPE_F16>(a, cut, as_stream(stream));
    default: return dispatch_rows<TGX_DTYPE_F32>(a, cut, as_stream(stream));
  }
}
