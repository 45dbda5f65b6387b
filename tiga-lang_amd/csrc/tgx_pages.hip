// Upkeep of a paged cache (Graph.append) and the choice of its pages a query
// row attends to (Graph.select_pages).
//
// append: sequence b's newest `queries` tokens, positions length - queries .. length - 1
// (those below zero do not exist), are rows b * queries + t of the new keys
// and values; each goes to its slot.  With page sums, every touched page's
// sum is formed again from the page's first row to its newest token, in fp32
// and in one order: a sum depends on what the page holds now and on nothing
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

// One workgroup per (sequence, touched page, kCells cells of N values of a
// row): kSlices threads share a cell, thread s taking the page's slots s, s +
// kSlices, ..., kBatch of them in flight at once; their sums are added in the
// order of s, so a page's sum is in one fixed order however its rows came in.
// Bound: memory for prompts (rows read and written once), latency for a
// single token.
constexpr int kCells = 32, kSlices = 8, kBatch = 4;

template <int DT, int N>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  using C = Cell<DT, N>;
  using T = typename C::T;
  using Raw = typename C::Raw;
  __shared__ float part[kSlices][kCells][N + 1];
  const PagedRel& r = a.rel;
  const int per_head = a.D / N, cells = a.heads * per_head;
  const int blocks = (cells + kCells - 1) / kCells;
  const int cell = blockIdx.x % blocks * kCells + threadIdx.x % kCells;
  const int slice = threadIdx.x / kCells;
  const int b = blockIdx.x / blocks / a.touched;
  const int length = paged_length(r, b);
  const int fresh = min(length, r.queries);        // new tokens that exist
  const int page = (length - fresh) / r.page_size + blockIdx.x / blocks % a.touched;
  if (fresh == 0 || page >= r.pages_per_seq) return;
  const int base = page * r.page_size;             // position of the page's first slot
  if (base >= length) return;
  const int id = r.table[b * r.seq_stride + page];
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(r.num_pages)) return;
  const int held = min(length - base, r.page_size);
  const int old = max(length - fresh - base, 0);   // slots filled before this call
  const int64_t slot0 = static_cast<int64_t>(id) * r.page_size;
  // Where the new row of the page's slot 0 would be.
  const int64_t row0 = static_cast<int64_t>(b) * r.queries + base - (length - r.queries);
  float s[N];
#pragma unroll
  for (int j = 0; j < N; ++j) s[j] = 0.f;
  const int h = cell / per_head, d = cell % per_head * N;
  if (cell < cells) {
    T* kc = static_cast<T*>(a.kc) + slot0 * a.kc_slot + h * a.kc_head + d;
    T* vc = static_cast<T*>(a.vc) + slot0 * a.vc_slot + h * a.vc_head + d;
    const T* k = static_cast<const T*>(a.k) + row0 * a.k_row + h * a.k_head + d;
    const T* v = static_cast<const T*>(a.v) + row0 * a.v_row + h * a.v_head + d;
    // Without sums the older slots are not read.
    const int first = a.sums ? slice : slice + (max(old - slice, 0) + kSlices - 1) / kSlices * kSlices;
    for (int o0 = first; o0 < held; o0 += kSlices * kBatch) {
      Raw kr[kBatch], vr[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int o = o0 + u * kSlices;
        if (o >= held) continue;
        kr[u] = C::load(o < old ? kc + o * a.kc_slot : k + o * a.k_row);
        if (o >= old) vr[u] = C::load(v + o * a.v_row);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int o = o0 + u * kSlices;
        if (o >= held) continue;
        if (o >= old) {
          C::store(kc + o * a.kc_slot, kr[u]);
          C::store(vc + o * a.vc_slot, vr[u]);
        }
        if (a.sums) C::add(kr[u], s);
      }
    }
  }
  if (!a.sums) return;
#pragma unroll
  for (int j = 0; j < N; ++j) part[slice][threadIdx.x % kCells][j] = s[j];
  __syncthreads();
  const int c = threadIdx.x / N, j = threadIdx.x % N;   // one value a thread
  const int out = blockIdx.x % blocks * kCells + c;
  if (c >= kCells || out >= cells) return;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < kSlices; ++w) sum += part[w][c][j];
  a.sums[(static_cast<int64_t>(id) * a.heads + out / per_head) * a.D + out % per_head * N + j] = sum;
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

// Whether the row's pages have to be ranked: fewer are wanted than there are.
__device__ __forceinline__ bool ranked(int pages, int count) { return count > 1 && pages > count; }

// Pages a workgroup of the scores covers: four waves, eight lanes a page, kUnroll
// pages a lane group.
constexpr int kUnroll = 4;
constexpr int kScorePages = 4 * 8 * kUnroll;

// Scores of kScorePages pages of one (row, head).  Eight lanes hold a page's
// D sums, 4 NJ values each, in 16-byte loads that make whole 128-byte lines;
// the lane's queries are summed over the group once, in fp64.  Bound: the
// page sums are read once, 4 D bytes a page and head; kUnroll pages' loads
// are issued before the first is used.
template <int DT, int NJ>
__global__ __launch_bounds__(256) void select_score_kernel(SelectArgs a) {
  using C = Cell<DT, 1>;
  const PagedRel& r = a.rel;
  const int pair = blockIdx.x % (a.heads * r.n_seqs * r.queries);   // heads fastest
  const int h = pair % a.heads, row = pair / a.heads;
  const int limit = row_limit(r, row);
  const int pages = (limit + r.page_size - 1) / r.page_size;
  const int page0 = (blockIdx.x / (a.heads * r.n_seqs * r.queries)) * kScorePages;
  if (!ranked(pages, a.count) || page0 >= pages - 1) return;
  const int lane = lane_id(), part = lane & 7, wave = threadIdx.x >> 6;
  const int32_t* ids = r.table + (row / r.queries) * r.seq_stride;
  int id[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int page = page0 + (wave * kUnroll + u) * 8 + (lane >> 3);
    id[u] = page < pages - 1 ? ids[page] : -1;
  }
  f32x4 s[kUnroll][NJ];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const bool named = static_cast<unsigned>(id[u]) < static_cast<unsigned>(r.num_pages);
    const float* p = a.sums + (static_cast<int64_t>(named ? id[u] : 0) * a.heads + h) * a.D;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int d = 4 * (8 * j + part);
      s[u][j] = d < a.D && named ? *reinterpret_cast<const f32x4*>(p + d)
                                 : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  const auto* q = static_cast<const typename C::T*>(a.q) + row * a.qs_row + h * a.qs_head;
  __shared__ __align__(16) double summed[32 * NJ];
  if (threadIdx.x < 32 * NJ) {
    const int d = threadIdx.x;
    double total = 0.0;
    for (int g = 0; d < a.D && g < a.group; ++g) {
      float f[1] = {0.f};
      C::add(C::load(q + g * a.qs_group + d), f);
      total += f[0];
    }
    summed[d] = total;
  }
  __syncthreads();
  double sum[NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[j][i] = summed[4 * (8 * j + part) + i];
  uint64_t* keys = a.keys + static_cast<int64_t>(pair) * r.pages_per_seq;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    double score = 0.0;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) score += sum[j][i] * static_cast<double>(s[u][j][i]);
#pragma unroll
    for (int mask = 1; mask < 8; mask <<= 1) score += __shfl_xor(score, mask, 64);
    if (static_cast<unsigned>(id[u]) >= static_cast<unsigned>(r.num_pages))
      score = -__builtin_huge_val();
    const int page = page0 + (wave * kUnroll + u) * 8 + (lane >> 3);
    if (part == 0 && page < pages - 1) keys[page] = ordered(score);
  }
}

// The same for widths the lanes do not hold: a thread per page.
template <int DT>
__global__ __launch_bounds__(256) void select_score_any_kernel(SelectArgs a, int64_t items) {
  using C = Cell<DT, 1>;
  const PagedRel& r = a.rel;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; item < items;
       item += static_cast<int64_t>(gridDim.x) * 256) {
    const int page = static_cast<int>(item % r.pages_per_seq);
    const int h = static_cast<int>(item / r.pages_per_seq % a.heads);
    const int row = static_cast<int>(item / r.pages_per_seq / a.heads);
    const int pages = (row_limit(r, row) + r.page_size - 1) / r.page_size;
    if (!ranked(pages, a.count) || page >= pages - 1) continue;
    const int id = r.table[(row / r.queries) * r.seq_stride + page];
    double score = -__builtin_huge_val();
    if (static_cast<unsigned>(id) < static_cast<unsigned>(r.num_pages)) {
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

// One workgroup per (row, head) takes the `want` largest of n keys.  A histogram
// of the keys' 16 leading bits (sign, exponent, four bits of the fraction),
// counted down from the largest key's, finds those of the want-th largest: among
// a few hundred or thousand scores, some twenty share them.  Where more than 64
// do, or the want-th lies further down, a histogram of each byte goes on (from
// the top).  The 64 or fewer that are left are ranked by a wave against each
// other, and (last, last_page) is the key and page of the want-th: a page is
// taken when its key is larger, or equal and the page no later.  A thread's
// first kHeld keys stay in registers.  Bound: latency, of some ten barriers.
constexpr int kHeld = 8;

template <int THREADS>
__global__ __launch_bounds__(THREADS) void select_pages_kernel(SelectArgs a) {
  constexpr int WAVES = THREADS / 64;
  const PagedRel& r = a.rel;
  __shared__ int hist[256];
  __shared__ int places[kHeld * WAVES];
  __shared__ int sh_bin, sh_left, sh_share, sh_n, sh_page;
  __shared__ uint64_t sh_last;
  __shared__ uint64_t cand[64];
  __shared__ int cand_page[64];
  const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
  const int h = blockIdx.x % a.heads;
  const int row = blockIdx.x / a.heads;
  const int limit = row_limit(r, row);
  const int pages = (limit + r.page_size - 1) / r.page_size;
  const int kept = min(pages, a.count);
  const int32_t* ids = r.table + (row / r.queries) * r.seq_stride;
  int32_t* out = a.table + static_cast<int64_t>(blockIdx.x) * a.count;
  const uint64_t* keys = a.keys + static_cast<int64_t>(blockIdx.x) * r.pages_per_seq;
  for (int i = kept + tid; i < a.count; i += THREADS) out[i] = -1;
  if (tid == 0 && h == 0)
    a.lengths[row] = kept ? (kept - 1) * r.page_size + limit - (pages - 1) * r.page_size : 0;
  if (kept == 0) return;
  const int n = pages - 1, want = kept - 1;
  if (!ranked(pages, a.count)) {
    if (kept == pages)
      for (int i = tid; i < pages; i += THREADS) out[i] = ids[i];
    else if (tid == 0)
      out[0] = ids[n];
    return;
  }
  if (tid == 0) out[want] = ids[n];
  uint64_t held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) held[j] = j * THREADS + tid < n ? keys[j * THREADS + tid] : 0;
  auto visit = [&](auto&& f) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j * THREADS + tid < n) f(j * THREADS + tid, held[j]);
    for (int i = kHeld * THREADS + tid; i < n; i += THREADS) f(i, keys[i]);
  };

  uint64_t prefix = 0, mask = 0;   // the leading bits settled so far
  int left = want;                 // rank of the want-th among the keys that share them
  int share = n;
  // Wave 0: the bin of hist (bins in descending order of key) that holds the
  // left-th largest; sh_share = 0 where the bins count too few.
  auto find = [&]() {
    if (wave != 0) return;
    int own[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += own[i] = hist[4 * lane + i];
    const int end = wave_prefix(sum);
    int above = end - sum;
    if (lane == 63 && end < left) sh_share = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (above < left && left <= above + own[i]) {
        sh_bin = 4 * lane + i;
        sh_left = left - above;
        sh_share = own[i];
      }
      above += own[i];
    }
  };
  int shift = 56;
  if (share > 64) {
    // The largest key's 16 leading bits (sign, exponent, four bits), and the 255
    // values below.
    uint32_t top = 0;
    visit([&](int, uint64_t key) { top = max(top, static_cast<uint32_t>(key >> 48)); });
    top = wave_largest(top);
    if (lane == 0) places[wave] = static_cast<int>(top);
    for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, static_cast<uint32_t>(places[w]));
    visit([&](int, uint64_t key) {
      const uint32_t bin = top - static_cast<uint32_t>(key >> 48);
      if (bin < 256) atomicAdd(&hist[bin], 1);
    });
    __syncthreads();
    find();
    __syncthreads();
    if (sh_share > 0) {
      prefix = static_cast<uint64_t>(top - sh_bin) << 48;
      mask = uint64_t{0xFFFF} << 48;
      left = sh_left;
      share = sh_share;
      shift = 40;
    }
  }
  for (; share > 64 && shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
    __syncthreads();
    visit([&](int, uint64_t key) {
      if ((key & mask) == prefix) atomicAdd(&hist[255 - (static_cast<int>(key >> shift) & 255)], 1);
    });
    __syncthreads();
    find();
    __syncthreads();
    prefix |= static_cast<uint64_t>(255 - sh_bin) << shift;
    mask |= uint64_t{255} << shift;
    left = sh_left;
    share = sh_share;
  }
  uint64_t last = prefix;
  int last_page = -1;    // -1: equal keys are counted off in order of position
  if (share <= 64) {
    if (tid == 0) sh_n = 0;
    __syncthreads();
    visit([&](int i, uint64_t key) {
      if ((key & mask) == prefix) {
        const int at = atomicAdd(&sh_n, 1);
        cand[at] = key;
        cand_page[at] = i;
      }
    });
    __syncthreads();
    if (wave == 0) {
      const uint64_t key = lane < share ? cand[lane] : 0;
      const int page = lane < share ? cand_page[lane] : 0;
      const int key_hi = static_cast<int>(key >> 32), key_lo = static_cast<int>(key);
      int rank = 0;
      for (int i = 0; i < share; ++i) {
        const uint64_t other =
            static_cast<uint64_t>(static_cast<uint32_t>(read_lane(key_hi, i))) << 32 |
            static_cast<uint32_t>(read_lane(key_lo, i));
        rank += other > key || (other == key && read_lane(page, i) < page);
      }
      if (lane < share && rank == left - 1) {
        sh_last = key;
        sh_page = page;
      }
    }
    __syncthreads();
    last = sh_last;
    last_page = sh_page;
  }
  // The taken pages in order of position: the ballots of kHeld * THREADS keys, one
  // scan of their counts, then every taken page's place.
  auto scan = [&](const unsigned long long (&set)[kHeld]) {
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) places[j * WAVES + wave] = __popcll(set[j]);
    }
    __syncthreads();
    if (wave == 0) {
      constexpr int EACH = (kHeld * WAVES + 63) / 64;
      int own[EACH], sum = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int at = EACH * lane + i;
        own[i] = at < kHeld * WAVES ? places[at] : 0;
        sum += own[i];
      }
      int before = wave_prefix(sum);
      if (lane == 63) sh_n = before;
      before -= sum;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int at = EACH * lane + i;
        if (at < kHeld * WAVES) places[at] = before;
        before += own[i];
      }
    }
    __syncthreads();
  };
  auto place = [&](unsigned long long set, int j) {
    return places[j * WAVES + wave] + __popcll(set & ((1ull << lane) - 1));
  };
  int placed = 0, seen = 0;
  for (int i0 = 0; i0 < n; i0 += kHeld * THREADS) {
    unsigned long long set[kHeld];
    if (i0 > 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        const int i = i0 + j * THREADS + tid;
        held[j] = i < n ? keys[i] : 0;
      }
    }
    unsigned counted = 0;   // bit j: the key is among the equal ones that are taken
    if (last_page < 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        set[j] = __ballot(i0 + j * THREADS + tid < n && held[j] == last);
      scan(set);
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (seen + place(set[j], j) < left) counted |= 1u << j;
      seen += sh_n;
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int i = i0 + j * THREADS + tid;
      const bool equal = last_page < 0 ? (counted >> j & 1) != 0 : i <= last_page;
      set[j] = __ballot(i < n && (held[j] > last || (held[j] == last && equal)));
    }
    scan(set);
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (set[j] >> lane & 1) out[placed + place(set[j], j)] = ids[i0 + j * THREADS + tid];
    placed += sh_n;
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int DT>
int launch_scores(const SelectArgs& a, hipStream_t s) {
  const int64_t pairs = static_cast<int64_t>(a.rel.n_seqs) * a.rel.queries * a.heads;
  const int64_t chunks = ceil_div(std::max(a.rel.pages_per_seq, 1), kScorePages);
  TGX_PROFILE("select_score", s);
  if (a.D % 4 == 0 && a.D <= 256 && aligned16(a.sums) && pairs * chunks <= kMaxBlocks256) {
    const dim3 grid(static_cast<uint32_t>(pairs * chunks));
    if (a.D <= 32) select_score_kernel<DT, 1><<<grid, dim3(256), 0, s>>>(a);
    else if (a.D <= 64) select_score_kernel<DT, 2><<<grid, dim3(256), 0, s>>>(a);
    else if (a.D <= 128) select_score_kernel<DT, 4><<<grid, dim3(256), 0, s>>>(a);
    else select_score_kernel<DT, 8><<<grid, dim3(256), 0, s>>>(a);
  } else {
    const int64_t items = pairs * a.rel.pages_per_seq;
    const dim3 grid(static_cast<uint32_t>(std::min(ceil_div(items, 256), kMaxBlocks256)));
    select_score_any_kernel<DT><<<grid, dim3(256), 0, s>>>(a, items);
  }
  TGX_LAUNCHED("select_score");
  return TGX_OK;
}

template <int DT>
int launch_append(const AppendArgs& a, bool vec, hipStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(a.rel.n_seqs) * a.touched *
                         ceil_div(static_cast<int64_t>(a.heads) * (vec ? a.D / 8 : a.D), kCells);
  TGX_REQUIRE(blocks <= kMaxBlocks256, "append: too many pages and heads for one launch");
  const dim3 grid(static_cast<uint32_t>(blocks));
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
  TGX_REQUIRE(p->n_seqs * p->queries * heads <= kMaxBlocks256 / 4,
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
  if (p->pages_per_seq > count && count > 1) {
    int st;
    switch (dtype) {
      case TGX_DTYPE_BF16: st = launch_scores<TGX_DTYPE_BF16>(a, s); break;
      case TGX_DTYPE_F16: st = launch_scores<TGX_DTYPE_F16>(a, s); break;
      default: st = launch_scores<TGX_DTYPE_F32>(a, s);
    }
    if (st) return st;
  }
  {
    TGX_PROFILE("select_pages", s);
    const dim3 grid(static_cast<uint32_t>(p->n_seqs * p->queries * heads));
    if (p->pages_per_seq <= 1024) select_pages_kernel<256><<<grid, dim3(256), 0, s>>>(a);
    else select_pages_kernel<1024><<<grid, dim3(1024), 0, s>>>(a);
  }
  TGX_LAUNCHED("select_pages");
  return TGX_OK;
}
