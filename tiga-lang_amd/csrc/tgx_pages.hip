// Upkeep of a paged cache (Graph.append) and the choice of its pages a query
// row attends to (Graph.select_pages).
//
// append: sequence b's newest `queries` tokens, positions length - queries .. length - 1
// (those below zero do not exist), are rows b * queries + t of the new keys
// and values; each goes to its slot.  With page sums, every touched page's
// sum is formed again from the page's first row to its newest token, in fp32
// and in slot order: a sum depends on what the page holds now and on nothing
// before it, so a program that takes tokens back and writes others keeps
// right sums.
//
// select: for each query row and key head, over the full pages p < n - 1 of
// the n = ceil(limit / page_size) that the row sees,
//
//   score_p = sum_d (sum_g q[row, h, g, d]) * page_sums[table[p], h, d]
//
// in fp64 (products of a 16-bit and a 32-bit value are exact there, and the
// choice turns on values next to each other); the count - 1 pages of largest
// score, equal scores to the lowest page, and the newest page, in order of
// position.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "tgx_device.h"
#include "tgx_host.h"
#include "tgx_paged.h"
#include "tgx_profile.h"
#include "tgx_vals.h"

namespace tgx {
namespace {

// ---------------------------------------------------------------------------
// append

struct AppendArgs {
  PagedRel rel;
  void* kc;
  void* vc;
  const void* k;
  const void* v;
  int64_t kc_slot, kc_head, vc_slot, vc_head;   // element strides
  int64_t k_row, k_head, v_row, v_head;
  float* sums;   // [num_pages, heads, D], may be null
  int heads, D;
  int touched;   // pages a sequence's new tokens lie on at most
};

// N consecutive values of one row; N = 1 for rows that are not on 16 bytes.
template <int DT, int N>
struct Cell {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  using Raw = typename V::Raw;
  static __device__ __forceinline__ Raw load(const T* p) { return V::load(p); }
  static __device__ __forceinline__ void store(T* p, Raw r) {
    *reinterpret_cast<Raw*>(p) = r;
  }
  static __device__ __forceinline__ void add(Raw r, float (&s)[N]) {
    float f[8];
    V::unpack(r, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += f[i];
  }
};
template <int DT>
struct Cell<DT, 1> {
  using T = typename Vals<DT, 8>::T;
  using Raw = T;
  static __device__ __forceinline__ Raw load(const T* p) { return *p; }
  static __device__ __forceinline__ void store(T* p, Raw r) { *p = r; }
  static __device__ __forceinline__ void add(Raw r, float (&s)[1]) {
    if constexpr (DT == TGX_DTYPE_F32) s[0] += r;
    else if constexpr (DT == TGX_DTYPE_BF16) s[0] += bf16_lo(r);
    else s[0] += static_cast<float>(__builtin_bit_cast(_Float16, r));
  }
};

// One workgroup per (sequence, touched page); a thread per N values of a row.
template <int DT, int N>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  using C = Cell<DT, N>;
  using T = typename C::T;
  const PagedRel& r = a.rel;
  const int b = blockIdx.x / a.touched;
  const int length = paged_length(r, b);
  const int fresh = min(length, r.queries);        // new tokens that exist
  const int page = (length - fresh) / r.page_size + blockIdx.x % a.touched;
  const int base = page * r.page_size;             // position of the page's first slot
  if (fresh == 0 || base >= length) return;
  const int id = r.table[b * r.seq_stride + page];
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(r.num_pages)) return;
  const int held = min(length - base, r.page_size);
  const int old = max(length - fresh - base, 0);   // slots filled before this call
  const int64_t slot0 = static_cast<int64_t>(id) * r.page_size;
  // New row of the page's slot `old`.
  const int64_t row0 = static_cast<int64_t>(b) * r.queries + (base + old) - (length - r.queries);
  const int per_head = a.D / N;
  for (int i = threadIdx.x; i < a.heads * per_head; i += 256) {
    const int h = i / per_head, d = i % per_head * N;
    T* kc = static_cast<T*>(a.kc) + slot0 * a.kc_slot + h * a.kc_head + d;
    T* vc = static_cast<T*>(a.vc) + slot0 * a.vc_slot + h * a.vc_head + d;
    const T* k = static_cast<const T*>(a.k) + row0 * a.k_row + h * a.k_head + d;
    const T* v = static_cast<const T*>(a.v) + row0 * a.v_row + h * a.v_head + d;
    float s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = 0.f;
    if (a.sums)
      for (int o = 0; o < old; ++o) C::add(C::load(kc + o * a.kc_slot), s);
    for (int o = old; o < held; ++o) {
      const typename C::Raw kr = C::load(k + (o - old) * a.k_row);
      C::store(kc + o * a.kc_slot, kr);
      C::store(vc + o * a.vc_slot, C::load(v + (o - old) * a.v_row));
      if (a.sums) C::add(kr, s);
    }
    if (a.sums) {
      float* dst = a.sums + (static_cast<int64_t>(id) * a.heads + h) * a.D + d;
#pragma unroll
      for (int j = 0; j < N; ++j) dst[j] = s[j];
    }
  }
}

// ---------------------------------------------------------------------------
// select

struct SelectArgs {
  PagedRel rel;
  const void* q;
  int64_t qs_row, qs_head, qs_group;
  const float* sums;     // [num_pages, heads, D] contiguous
  int heads, group, D;
  int count;
  int32_t* table;        // [rows, heads, count]
  int32_t* lengths;      // [rows]
  uint64_t* keys;        // [rows, heads, pages_per_seq] ordered scores
};

// Positions that row b * queries + t sees.
__device__ __forceinline__ int row_limit(const PagedRel& r, int row) {
  const int b = row / r.queries, t = row % r.queries;
  return max(paged_length(r, b) - (r.queries - 1 - t), 0);
}

// A score as an unsigned number of the same order; NaN as -inf.
__device__ __forceinline__ uint64_t ordered(double s) {
  if (s != s) s = -__builtin_huge_val();
  if (s == 0.0) s = 0.0;   // -0 and +0 are equal scores
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(s));
  return u >> 63 ? ~u : u | (uint64_t{1} << 63);
}

// One thread per (row, head, full page): the whole dot product.
template <int DT>
__global__ __launch_bounds__(256) void select_score_kernel(SelectArgs a, int64_t items) {
  const PagedRel& r = a.rel;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; item < items;
       item += static_cast<int64_t>(gridDim.x) * 256) {
    const int page = static_cast<int>(item % r.pages_per_seq);
    const int h = static_cast<int>(item / r.pages_per_seq % a.heads);
    const int row = static_cast<int>(item / r.pages_per_seq / a.heads);
    const int limit = row_limit(r, row);
    if (page >= (limit + r.page_size - 1) / r.page_size - 1) continue;
    const int id = r.table[(row / r.queries) * r.seq_stride + page];
    double score = -__builtin_huge_val();
    if (static_cast<unsigned>(id) < static_cast<unsigned>(r.num_pages)) {
      using C = Cell<DT, 1>;
      const auto* q = static_cast<const typename C::T*>(a.q) + row * a.qs_row + h * a.qs_head;
      const float* s = a.sums + (static_cast<int64_t>(id) * a.heads + h) * a.D;
      score = 0.0;
      for (int d = 0; d < a.D; ++d) {
        double sum = 0.0;
        for (int g = 0; g < a.group; ++g) {
          float f[1] = {0.f};
          C::add(C::load(q + g * a.qs_group + d), f);
          sum += f[0];
        }
        score += sum * s[d];
      }
    }
    a.keys[item] = ordered(score);
  }
}

// Rank of this thread among the workgroup's threads with `flag` set, and their number.
__device__ __forceinline__ int block_rank(bool flag, int* wave_counts, int& total) {
  const unsigned long long set = __ballot(flag);
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) wave_counts[wave] = __popcll(set);
  __syncthreads();
  int before = __popcll(set & ((1ull << lane) - 1));
  total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) before += wave_counts[w];
    total += wave_counts[w];
  }
  return before;
}

// One workgroup per (row, head): the want-th largest key byte by byte from
// the top, then the chosen pages in order of position.
__global__ __launch_bounds__(256) void select_pages_kernel(SelectArgs a) {
  const PagedRel& r = a.rel;
  __shared__ int hist[256];
  __shared__ int wave_counts[4];
  __shared__ uint64_t sh_prefix;
  __shared__ int sh_want;
  const int h = blockIdx.x % a.heads;
  const int row = blockIdx.x / a.heads;
  const int limit = row_limit(r, row);
  const int pages = (limit + r.page_size - 1) / r.page_size;
  const int kept = min(pages, a.count);
  const int32_t* ids = r.table + (row / r.queries) * r.seq_stride;
  int32_t* out = a.table + static_cast<int64_t>(blockIdx.x) * a.count;
  const uint64_t* keys = a.keys + static_cast<int64_t>(blockIdx.x) * r.pages_per_seq;
  for (int i = kept + threadIdx.x; i < a.count; i += 256) out[i] = -1;
  if (threadIdx.x == 0 && h == 0)
    a.lengths[row] = kept ? (kept - 1) * r.page_size + limit - (pages - 1) * r.page_size : 0;
  if (kept == 0) return;
  if (threadIdx.x == 0) out[kept - 1] = ids[pages - 1];
  const int n = pages - 1, want = kept - 1;
  if (want == n) {
    for (int i = threadIdx.x; i < n; i += 256) out[i] = ids[i];
    return;
  }
  if (want == 0) return;
  // Radix select: after each byte, `prefix` holds the want-th largest key's
  // leading bytes and sh_want its rank among the keys that share them.
  if (threadIdx.x == 0) {
    sh_prefix = 0;
    sh_want = want;
  }
  for (int shift = 56; shift >= 0; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t prefix = sh_prefix;
    for (int i = threadIdx.x; i < n; i += 256) {
      const uint64_t key = keys[i];
      if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = sh_want, byte = 255;
      while (hist[byte] < left) left -= hist[byte--];
      sh_want = left;
      sh_prefix = prefix | (static_cast<uint64_t>(byte) << shift);
    }
    __syncthreads();
  }
  const uint64_t last = sh_prefix;
  const int equal = sh_want;   // of the pages with this score, the first so many
  int placed = 0, seen = 0;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + threadIdx.x;
    const uint64_t key = i < n ? keys[i] : 0;
    const bool tie = i < n && key == last;
    int ties, taken;
    const int tie_rank = block_rank(tie, wave_counts, ties);
    const bool take = i < n && (key > last || (tie && seen + tie_rank < equal));
    const int at = block_rank(take, wave_counts, taken);
    if (take) out[placed + at] = ids[i];
    placed += taken;
    seen += ties;
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int DT>
int launch_append(const AppendArgs& a, bool vec, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(static_cast<int64_t>(a.rel.n_seqs) * a.touched));
  {
    TGX_PROFILE("paged_append", stream);
    if (vec) append_kernel<DT, 8><<<grid, dim3(256), 0, stream>>>(a);
    else append_kernel<DT, 1><<<grid, dim3(256), 0, stream>>>(a);
  }
  TGX_LAUNCHED("paged_append");
  return TGX_OK;
}

int check_select(const tgx_paged* p, int heads, int group, int D, int count) {
  if (int st = check_paged(p)) return st;
  TGX_REQUIRE(p->table_heads == 1, "pages are selected from one table per sequence");
  TGX_REQUIRE(heads >= 1 && group >= 1 && D >= 1 && count >= 1,
              "heads, group, head width and count must be positive");
  TGX_REQUIRE(p->n_seqs * p->queries * heads <= kMaxBlocks256,
              "page selection: too many rows and heads for one launch");
  return TGX_OK;
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_paged_append(const tgx_paged* p, void* key_cache_dev, const void* key_dev,
                                void* value_cache_dev, const void* value_dev,
                                const int64_t* strides, float* page_sums_dev, int heads, int D,
                                int dtype, void* stream) {
  if (int st = check_paged(p)) return st;
  TGX_REQUIRE(p->table_heads == 1, "rows are appended through one table per sequence");
  TGX_REQUIRE(heads >= 1 && D >= 1, "heads and head width must be positive");
  TGX_REQUIRE(dtype_bytes(dtype) != 0, "unknown dtype %d", dtype);
  if (p->n_seqs == 0 || p->num_pages == 0 || p->pages_per_seq == 0) return TGX_OK;
  TGX_REQUIRE(key_cache_dev && key_dev && value_cache_dev && value_dev && strides,
              "null operand");
  // Pages that `queries` consecutive positions can lie on, of those the table has.
  const int64_t touched = std::min<int64_t>((p->queries - 1) / p->page_size + 2,
                                            p->pages_per_seq);
  TGX_REQUIRE(p->n_seqs * touched <= kMaxBlocks256, "append: too many pages for one launch");
  AppendArgs a{};
  a.rel = paged_rel(*p);
  a.kc = key_cache_dev;
  a.vc = value_cache_dev;
  a.k = key_dev;
  a.v = value_dev;
  a.kc_slot = strides[0], a.kc_head = strides[1];
  a.k_row = strides[2], a.k_head = strides[3];
  a.vc_slot = strides[4], a.vc_head = strides[5];
  a.v_row = strides[6], a.v_head = strides[7];
  a.sums = page_sums_dev;
  a.heads = heads;
  a.D = D;
  a.touched = static_cast<int>(touched);
  const int vec = 16 / dtype_bytes(dtype);
  bool wide = D % 8 == 0 && aligned16(key_cache_dev) && aligned16(key_dev) &&
              aligned16(value_cache_dev) && aligned16(value_dev);
  for (int i = 0; i < 8; ++i) wide = wide && strides[i] % vec == 0;
  switch (dtype) {
    case TGX_DTYPE_BF16: return launch_append<TGX_DTYPE_BF16>(a, wide, as_stream(stream));
    case TGX_DTYPE_F16: return launch_append<TGX_DTYPE_F16>(a, wide, as_stream(stream));
    default: return launch_append<TGX_DTYPE_F32>(a, wide, as_stream(stream));
  }
}

extern "C" int tgx_select_pages_workspace(const tgx_paged* p, int heads, int count,
                                          size_t* bytes) {
  TGX_REQUIRE(bytes != nullptr, "null bytes");
  if (int st = check_select(p, heads, 1, 1, count)) return st;
  *bytes = sizeof(uint64_t) * p->n_seqs * p->queries * heads * p->pages_per_seq;
  return TGX_OK;
}

extern "C" int tgx_select_pages(const tgx_paged* p, const void* q_dev, const int64_t* strides,
                                const float* page_sums_dev, int heads, int group, int D,
                                int dtype, int count, int32_t* table_dev, int32_t* lengths_dev,
                                void* workspace_dev, size_t workspace_bytes, void* stream) {
  if (int st = check_select(p, heads, group, D, count)) return st;
  TGX_REQUIRE(dtype_bytes(dtype) != 0, "unknown dtype %d", dtype);
  if (p->n_seqs == 0) return TGX_OK;
  TGX_REQUIRE(q_dev && strides && table_dev && lengths_dev, "null operand");
  TGX_REQUIRE(p->num_pages == 0 || page_sums_dev, "null page sums");
  size_t need = 0;
  if (int st = tgx_select_pages_workspace(p, heads, count, &need)) return st;
  TGX_REQUIRE(workspace_bytes >= need && (need == 0 || workspace_dev),
              "workspace of %zu bytes, needs %zu", workspace_bytes, need);
  SelectArgs a{};
  a.rel = paged_rel(*p);
  a.q = q_dev;
  a.qs_row = strides[0], a.qs_head = strides[1], a.qs_group = strides[2];
  a.sums = page_sums_dev;
  a.heads = heads;
  a.group = group;
  a.D = D;
  a.count = count;
  a.table = table_dev;
  a.lengths = lengths_dev;
  a.keys = static_cast<uint64_t*>(workspace_dev);
  hipStream_t s = as_stream(stream);
  const int64_t pairs = p->n_seqs * p->queries * heads;
  const int64_t items = pairs * p->pages_per_seq;
  if (items > 0) {
    const dim3 grid(static_cast<uint32_t>(std::min(ceil_div(items, 256), kMaxBlocks256)));
    TGX_PROFILE("select_score", s);
    switch (dtype) {
      case TGX_DTYPE_BF16:
        select_score_kernel<TGX_DTYPE_BF16><<<grid, dim3(256), 0, s>>>(a, items);
        break;
      case TGX_DTYPE_F16:
        select_score_kernel<TGX_DTYPE_F16><<<grid, dim3(256), 0, s>>>(a, items);
        break;
      default: select_score_kernel<TGX_DTYPE_F32><<<grid, dim3(256), 0, s>>>(a, items);
    }
  }
  TGX_LAUNCHED("select_score");
  {
    TGX_PROFILE("select_pages", s);
    select_pages_kernel<<<dim3(static_cast<uint32_t>(pairs)), dim3(256), 0, s>>>(a);
  }
  TGX_LAUNCHED("select_pages");
  return TGX_OK;
}
