// Attention over a paged relation (Graph.paged) whose cache has the queries' type:
// the launches of tgx_paged_attn.h's kernels, and the entry points.
#include "tgx_paged_attn.h"

namespace tgx {
namespace {

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

// Tiles a sequence's rows see at most.
int64_t most_tiles(const tgx_paged& p, const tgx_paged_view& w) {
  const int64_t positions = static_cast<int64_t>(p.pages_per_seq) * p.page_size;
  int64_t tiles = ceil_div(positions, kTile);
  if (w.window > 0)   // (a run of n positions lies on n / 64 + 2 tiles at most)
    tiles = std::min(tiles, ceil_div(std::min<int64_t>(w.sinks, positions), kTile) +
                                (static_cast<int64_t>(w.window) + p.queries - 1) / kTile + 2);
  return tiles;
}

Cut cut_of(const tgx_paged& p, const tgx_paged_view& w, int heads, int group, int D, int dtype) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  const int held = held_queries(p, group, D, dtype);
  const int64_t each = workgroups_per_piece(p, heads, group, D, dtype);
  const int64_t tiles = most_tiles(p, w);
  // Windowed and 8-bit tiles of up to 16 queries take the workgroups that are resident at
  // once (their registers allow two, three and four a CU), so that a launch is one round
  // of equal pieces (64 sequences of 100-4000, 8 bits: 81 us with four a CU at
  // D = 128, 77 us with two; 4 of 100k-131k: 186-197 us with three, six or eight, 184
  // with two); those of 16-bit caches without a window came out as they were.
  const bool by_heads = held == 16 && (w.code != 0 || w.window > 0);
  const int per_cu = held > 64 ? 2 : !by_heads ? 4 : D == 128 ? 2 : D == 64 ? 3 : 4;
  const int64_t wanted = cus * per_cu / each;
  const int64_t queries = static_cast<int64_t>(p.table_heads) * heads * p.queries * group;
  if (tiles <= kMinTiles || wanted <= 1 || p.n_seqs > kMaxBlocks256 / queries ||
      (tiles <= kWholeTiles && p.n_seqs * each >= cus))
    return Cut{1, p.n_seqs, false};
  Cut cut{wanted, 0, true};
  // Workgroups of several heads, pieces of as many tiles a wave, and as many
  // workgroups, as of one; not where the smallest pieces of all sequences are
  // resident at once: the time is one of latency there, and more pieces to join
  // (8 sequences that see 1088 keys, 8 heads: 14.8 us with one head, 17.8 with four).
  const bool few = p.n_seqs * ceil_div(tiles, kMinTiles) * each <= int64_t{cus} * per_cu;
  if (by_heads && !few) cut.heads_held = heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
  cut.wanted *= cut.heads_held;
  cut.min_tiles = kMinTiles / cut.heads_held;
  cut.launched = std::min(cut.wanted + p.n_seqs, p.n_seqs * ceil_div(tiles, cut.min_tiles));
  return cut;
}

int check_attn(const tgx_paged* p, const tgx_paged_view& w, int heads, int group, int D,
               int dtype) {
  if (int st = check_paged(p)) return st;
  TGX_REQUIRE(w.window >= 0 && w.sinks >= 0 && (w.window > 0 || w.sinks == 0),
              "window and sinks must not be negative, and sinks need a window");
  TGX_REQUIRE(w.code == 0 || known_code(w.code), "unknown code %d", w.code);
  TGX_REQUIRE(w.code == 0 || (w.block >= 1 && p->page_size % w.block == 0),
              "pages of %d slots are no whole blocks of %d", p->page_size, w.block);
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
      cut_of(*p, w, heads, group, D, dtype).launched > kMaxBlocks256 / each - 8) {
    set_error("paged attention: too many sequences, heads and queries for one launch");
    return TGX_UNSUPPORTED;
  }
  return TGX_OK;
}

size_t meta_bytes(const tgx_paged& p) { return align_up(sizeof(int2) * p.n_seqs); }

template <int DT, int LPK, bool WIN>
int launch_rows(const PagedArgs& a, const Cut& cut, hipStream_t stream) {
  const int64_t queries = static_cast<int64_t>(a.rel.heads) * a.heads * a.rel.queries * a.group;
  TGX_PROFILE("paged_rows", stream);
  paged_rows_kernel<DT, LPK, 0, WIN>
      <<<dim3(static_cast<uint32_t>(cut.launched * queries)), dim3(256), 0, stream>>>(a);
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

template <int DT, bool WIN>
int dispatch_rows(const PagedArgs& a, const Cut& cut, hipStream_t stream) {
  if (a.D <= 32) return launch_rows<DT, 4, WIN>(a, cut, stream);
  if (a.D <= 64) return launch_rows<DT, 8, WIN>(a, cut, stream);
  if (a.D <= 128) return launch_rows<DT, 16, WIN>(a, cut, stream);
  if (a.D <= 256) return launch_rows<DT, 32, WIN>(a, cut, stream);
  return launch_rows<DT, 64, WIN>(a, cut, stream);
}

template <int DT>
int dispatch_join(const PagedArgs& a, hipStream_t stream) {
  if (a.D <= 32) return launch_join<DT, 4>(a, stream);
  if (a.D <= 64) return launch_join<DT, 8>(a, stream);
  if (a.D <= 128) return launch_join<DT, 16>(a, stream);
  if (a.D <= 256) return launch_join<DT, 32>(a, stream);
  return launch_join<DT, 64>(a, stream);
}

template <typename T, int D, bool WIN>
int launch_tiles(const PagedArgs& a, const Cut& cut, int held, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.rel.queries) * a.group;
  const int64_t pieces = cut.launched * a.rel.heads * a.heads;
  TGX_PROFILE("paged_tiles", stream);
  if (held == 16) {
    const int64_t blocks =
        WIN ? ceil_div(cut.launched, 8) * 8 * a.rel.heads * a.heads / a.held : pieces;
    paged_tile_kernel<T, D, WIN><<<dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream>>>(a);
  } else {
    const dim3 grid(static_cast<uint32_t>(ceil_div(pieces, 8) * 8 * ceil_div(rows, held)));
    if (held == 32) paged_block_kernel<T, D, 2, 1, 0, WIN><<<grid, dim3(256), 0, stream>>>(a);
    else if (held == 64) paged_block_kernel<T, D, 1, 1, 0, WIN><<<grid, dim3(256), 0, stream>>>(a);
    else paged_block_kernel<T, D, 1, 2, 0, WIN><<<grid, dim3(256), 0, stream>>>(a);
  }
  TGX_LAUNCHED("paged_tiles");
  return TGX_OK;
}

template <typename T, bool WIN>
int dispatch_tiles(const PagedArgs& a, const Cut& cut, int held, hipStream_t stream) {
  if (a.D == 32) return launch_tiles<T, 32, WIN>(a, cut, held, stream);
  if (a.D == 64) return launch_tiles<T, 64, WIN>(a, cut, held, stream);
  return launch_tiles<T, 128, WIN>(a, cut, held, stream);
}

// The launches over caches of the queries' type, without the join.
template <bool WIN>
int dispatch_whole(const PagedArgs& a, const Cut& cut, bool tiles, int held, int dtype,
                   hipStream_t s) {
  switch (dtype) {
    case TGX_DTYPE_BF16:
      return tiles ? dispatch_tiles<__bf16, WIN>(a, cut, held, s)
                   : dispatch_rows<TGX_DTYPE_BF16, WIN>(a, cut, s);
    case TGX_DTYPE_F16:
      return tiles ? dispatch_tiles<_Float16, WIN>(a, cut, held, s)
                   : dispatch_rows<TGX_DTYPE_F16, WIN>(a, cut, s);
    default:
      return dispatch_rows<TGX_DTYPE_F32, WIN>(a, cut, s);
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace tgx

using namespace tgx;

static int attn_workspace(const tgx_paged* p, const tgx_paged_view& w, int heads, int group, int D,
                          int dtype, size_t* bytes) {
  TGX_REQUIRE(bytes != nullptr, "null bytes");
  if (int st = check_attn(p, w, heads, group, D, dtype)) return st;
  const int64_t groups = static_cast<int64_t>(p->table_heads) * heads;
  const Cut cut = cut_of(*p, w, heads, group, D, dtype);
  *bytes = !cut.split ? 0
                      : meta_bytes(*p) + sizeof(float) * cut.launched * groups * group *
                                             p->queries * (D + 2);
  return TGX_OK;
}

static int attn(const tgx_paged* p, const tgx_paged_view& w, const void* q_dev, const void* k_dev,
                const void* v_dev, const int64_t* strides, float scale, void* out_dev, int heads,
                int group, int D, int dtype, void* workspace_dev, size_t workspace_bytes,
                void* stream) {
  if (int st = check_attn(p, w, heads, group, D, dtype)) return st;
  if (p->n_seqs == 0) return TGX_OK;
  TGX_REQUIRE(q_dev && out_dev && strides, "null operand");
  TGX_REQUIRE(p->num_pages == 0 || (k_dev && v_dev), "null cache");
  TGX_REQUIRE(p->num_pages == 0 || w.code == 0 || (w.k_scales_dev && w.v_scales_dev),
              "null scales");
  TGX_REQUIRE(aligned16(q_dev) && aligned16(out_dev), "q and out must start on 16 bytes");
  // Values of a 16-byte load; codes are read by eights where their rows do not allow more.
  const int vec = 16 / dtype_bytes(dtype);
  bool sixteens = aligned16(k_dev) && aligned16(v_dev);
  TGX_REQUIRE(w.code != 0 || sixteens, "k and v must start on 16 bytes");
  TGX_REQUIRE(reinterpret_cast<uintptr_t>(k_dev) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(v_dev) % 8 == 0,
              "codes must start on 8 bytes");
  for (int i = 0; i < 9; ++i) {
    const int by = i < 3 || w.code == 0 ? vec : 8;
    TGX_REQUIRE(strides[i] % by == 0, "stride %lld does not keep rows on %d bytes",
                static_cast<long long>(strides[i]), i < 3 || w.code == 0 ? 16 : 8);
    if (i >= 3 && strides[i] % 16 != 0) sixteens = false;
  }
  size_t need = 0;
  if (int st = attn_workspace(p, w, heads, group, D, dtype, &need)) return st;
  TGX_REQUIRE(workspace_bytes >= need && (need == 0 || workspace_dev),
              "workspace of %zu bytes, needs %zu", workspace_bytes, need);
  const Cut cut = cut_of(*p, w, heads, group, D, dtype);
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
  a.min_tiles = cut.min_tiles;
  a.held = cut.heads_held;
  if (cut.split) {
    a.meta = static_cast<int2*>(workspace_dev);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace_dev) + meta_bytes(*p));
  }
  // A window of all that a table holds hides nothing.
  const int positions = p->pages_per_seq * p->page_size;
  a.window = w.window > 0 ? std::min(w.window, positions) : positions;
  a.sinks = std::min(w.sinks, positions);
  a.k_scales = w.k_scales_dev;
  a.v_scales = w.v_scales_dev;
  a.block = static_cast<unsigned>(std::max(w.block, 1));
  hipStream_t s = as_stream(stream);
  const bool tiles = tiled(D, dtype);
  const int held = held_queries(*p, group, D, dtype);
  int st;
  if (w.code != 0)
    // (A workgroup's queries are the same on either kernel: the cut holds.)
    st = paged_attn_scaled(a, cut, tiles && sixteens ? held : 0, dtype, w.code, s);
  else if (w.window > 0)
    st = dispatch_whole<true>(a, cut, tiles, held, dtype, s);
  else
    st = dispatch_whole<false>(a, cut, tiles, held, dtype, s);
  if (st || !cut.split) return st;
  switch (dtype) {
    case TGX_DTYPE_BF16: return dispatch_join<TGX_DTYPE_BF16>(a, s);
    case TGX_DTYPE_F16: return dispatch_join<TGX_DTYPE_F16>(a, s);
    default: return dispatch_join<TGX_DTYPE_F32>(a, s);
  }
}

extern "C" int tgx_paged_attn_workspace(const tgx_paged* p, int heads, int group, int D,
                                        int dtype, size_t* bytes) {
  return attn_workspace(p, tgx_paged_view{}, heads, group, D, dtype, bytes);
}

extern "C" int tgx_paged_attn(const tgx_paged* p, const void* q_dev, const void* k_dev,
                              const void* v_dev, const int64_t* strides, float scale,
                              void* out_dev, int heads, int group, int D, int dtype,
                              void* workspace_dev, size_t workspace_bytes, void* stream) {
  return attn(p, tgx_paged_view{}, q_dev, k_dev, v_dev, strides, scale, out_dev, heads, group, D,
              dtype, workspace_dev, workspace_bytes, stream);
}

extern "C" int tgx_paged_attn_view_workspace(const tgx_paged* p, const tgx_paged_view* view,
                                             int heads, int group, int D, int dtype,
                                             size_t* bytes) {
  TGX_REQUIRE(view != nullptr, "null view");
  return attn_workspace(p, *view, heads, group, D, dtype, bytes);
}

extern "C" int tgx_paged_attn_view(const tgx_paged* p, const tgx_paged_view* view,
                                   const void* q_dev, const void* k_dev, const void* v_dev,
                                   const int64_t* strides, float scale, void* out_dev, int heads,
                                   int group, int D, int dtype, void* workspace_dev,
                                   size_t workspace_bytes, void* stream) {
  TGX_REQUIRE(view != nullptr, "null view");
  return attn(p, *view, q_dev, k_dev, v_dev, strides, scale, out_dev, heads, group, D, dtype,
              workspace_dev, workspace_bytes, stream);
}
