// Upkeep of a paged cache held in 8 bits (Graph.append on tiga.BlockScaled) and
// reading it back (Graph.read).
//
// append: the newest tokens' rows x of a block of `block` slots, for each head, with
// M the largest code:
//
//   s' = the smallest power of two >= 2^-126 with max |x| <= M s'
//   s  = the scale s_old of the block's older tokens where s' <= |s_old|, else s'
//        (s' where there are none)
//   code = rne(x / s);  an older token's code = rne(code * s_old / s)
//
// x / s is exact for a power of two, so a code is the definition's whatever the
// arithmetic; a scale that stays leaves the older codes as they are, and one that
// grows shifts them.  A NaN or an infinity among x makes s NaN: codes cannot hold
// them, and what they touch must not read back as numbers.  With page sums, every
// touched page's sum of code * s over its slots up to the newest token is formed
// again, in fp32 and in one order.
//
// read: rows of code * s, rounded once.
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
namespace {

struct ScaledAppendArgs {
  PagedRel rel;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;             // [slots / block, heads]
  float* vs;
  const void* k;
  const void* v;
  int64_t kc_slot, kc_head, vc_slot, vc_head;   // elements
  int64_t k_row, k_head, v_row, v_head;
  float* sums;           // [num_pages, heads, D], may be null
  int heads, D, block;
  int touched;           // pages a sequence's new tokens lie on at most
};

// One workgroup per (sequence, touched page, head), two waves for the keys and two for
// the values, which take the page's blocks in turn; of pages of one block, a
// workgroup per two heads.  LPR lanes hold a row, 8 values each, and a wave takes 64 /
// LPR rows at a time, kHold times of them in flight and kept until the scale is known
// (of longer blocks the rest is read again, from the caches).
// Bound: memory for prompts (16-bit rows read, codes written: 8 of 1500 tokens, 16
// heads of 64, 15 us), latency for a single token (64 sequences: 5.2 us).  One pass over the
// rows instead of two, codes by one product and one fused add, and keys and values on
// waves of their own took those prompts, written and read back, from 58 to 32 us.
constexpr int kHold = 4;

template <int DT, int LPR, int CODE>
__global__ __launch_bounds__(256) void append_scaled_kernel(ScaledAppendArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  constexpr int RPI = 64 / LPR;
  __shared__ float part[2][RPI][LPR * 8];
  const PagedRel& r = a.rel;
  const bool pair = r.page_size == a.block;      // two heads a workgroup
  const int groups = pair ? (a.heads + 1) / 2 : a.heads;
  // A page's heads are workgroups 8 apart, on one XCD's L2: they write parts of its lines.
  const int of8 = blockIdx.x / 8, group = of8 % groups;
  const int item = of8 / groups * 8 + blockIdx.x % 8;
  const int b = item / a.touched;
  if (b >= r.n_seqs) return;
  const int length = paged_length(r, b);
  const int fresh = min(length, r.queries);        // new tokens that exist
  const int page = (length - fresh) / r.page_size + item % a.touched;
  if (fresh == 0 || page >= r.pages_per_seq) return;
  const int base = page * r.page_size;             // position of the page's first slot
  if (base >= length) return;
  const int id = r.table[b * r.seq_stride + page];
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(r.num_pages)) return;
  const int held = min(length - base, r.page_size);
  const int old = max(length - fresh - base, 0);   // slots filled before this call
  const int64_t slot0 = static_cast<int64_t>(id) * r.page_size;
  const int64_t row0 = static_cast<int64_t>(b) * r.queries + base - (length - r.queries);
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int half = wave >> 1;
  const bool keys = (wave & 1) == 0, sums = keys && a.sums;
  const int h = pair ? group * 2 + half : group;
  const int sub = lane / LPR, d = lane % LPR * 8;
  const bool has = d < a.D;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.f;

  if (h < a.heads) {
    const int64_t c_slot = keys ? a.kc_slot : a.vc_slot, x_row = keys ? a.k_row : a.v_row;
    uint8_t* cb = (keys ? a.kc : a.vc) + slot0 * c_slot + h * (keys ? a.kc_head : a.vc_head) + d;
    const T* xb = static_cast<const T*>(keys ? a.k : a.v) + row0 * x_row +
                  h * (keys ? a.k_head : a.v_head) + d;
    float* scales = (keys ? a.ks : a.vs) + slot0 / a.block * a.heads + h;
    const int first = sums ? 0 : old / a.block, step = pair ? 1 : 2;
    for (int j = pair ? first : first + ((first ^ half) & 1); j * a.block < held; j += step) {
      const int s0 = j * a.block, s1 = min(s0 + a.block, held);
      const int from = min(max(old, s0), s1);        // the block's first new slot
      float* at = scales + static_cast<int64_t>(j) * a.heads;
      float scale = from > s0 ? *at : 0.f;
      const float before = scale;
      // The lane's first new slot: slot s0 + sub + k RPI is always its own, so that
      // sums are in one order however the rows came in.
      const int begin = s0 + sub + (max(from - s0 - sub, 0) + RPI - 1) / RPI * RPI;
      typename V::Raw x[kHold];
      if (from < s1) {
        Magnitude<DT> top;
        for (int s = begin + kHold * RPI; has && s < s1; s += RPI) top.see(V::load(xb + s * x_row));
#pragma unroll
        for (int u = 0; u < kHold; ++u)
          x[u] = has && begin + u * RPI < s1 ? V::load(xb + (begin + u * RPI) * x_row)
                                             : typename V::Raw{};
#pragma unroll
        for (int u = 0; u < kHold; ++u) top.see(x[u]);
        const float need = block_scale<CODE>(wave_largest(top.bits()));
        // By magnitude: a scale from elsewhere may be negative.  (Either one's NaN stays.)
        scale = from == s0 || !(need <= fabsf(scale)) ? (scale != scale ? scale : need) : scale;
        if (lane == 0) *at = scale;
      }
      const bool lost = scale != scale;
      auto add = [&](u32x2 w) {
        float f[8];
        widen8<CODE>(w, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += f[i] * scale;
      };
      // The older tokens, by the new scale.
      const bool again = from > s0 && from < s1 && scale != before && !lost;
      if ((sums || again) && has) {
        const float ratio = again ? before / scale : 1.f;
        for (int s = s0 + sub; s < from; s += RPI) {
          u32x2 w = *reinterpret_cast<const u32x2*>(cb + s * c_slot);
          if (again) {
            float f[8];
            widen8<CODE>(w, f);
            w = encode8<CODE>(f, ratio);
            *reinterpret_cast<u32x2*>(cb + s * c_slot) = w;
          }
          if (sums) add(w);
        }
      }
      // By a power of two the quotient is a product; by a scale that the block had from
      // elsewhere it is divided.
      const bool power = (__float_as_uint(scale) & 0x7FFFFFu) == 0;
      const float by = power ? 1.f / scale : 1.f;
      auto put = [&](int s, const typename V::Raw& raw) {
        u32x2 w = {0u, 0u};
        if (!lost) {
          float f[8];
          V::unpack(raw, f);
          if (!power) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = f[i] / scale;
          }
          w = encode8<CODE>(f, by);
        }
        *reinterpret_cast<u32x2*>(cb + s * c_slot) = w;
        if (sums) add(w);
      };
      if (from < s1 && has) {
#pragma unroll
        for (int u = 0; u < kHold; ++u)
          if (begin + u * RPI < s1) put(begin + u * RPI, x[u]);
        for (int s = begin + kHold * RPI; s < s1; s += RPI) put(s, V::load(xb + s * x_row));
      }
    }
  }
  if (!a.sums) return;
  if (keys) {
#pragma unroll
    for (int i = 0; i < 8; ++i) part[half][sub][d + i] = sum[i];
  }
  __syncthreads();
  const int page_heads = pair ? 2 : 1;
  for (int c = threadIdx.x; c < page_heads * a.D; c += 256) {
    const int which = c / a.D, e = c % a.D;
    const int head = pair ? group * 2 + which : h;
    if (head >= a.heads) continue;
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < RPI; ++w) total += part[which][w][e];
    if (!pair) {
#pragma unroll
      for (int w = 0; w < RPI; ++w) total += part[1][w][e];
    }
    a.sums[(static_cast<int64_t>(id) * a.heads + head) * a.D + e] = total;
  }
}

// Below this many workgroups of four parts a thread one part each fills more of the
// GPU; and what is written is stored past the caches from this size on.  8 heads of 128,
// e4m3 to bf16, calls of a graph one after another: rows (workgroups of four parts, bytes
// written) and us with one part a thread, with four, and with four past the caches:
//   256 (32, 1 MB)        3.6    7.4    7.4       16384 (2048, 64 MB)   19.9   22.2   20.3
//   4096 (512, 16 MB)     7.7   10.0    8.7       64000 (8000, 250 MB)  95     90     62
//   8192 (1024, 32 MB)   12.4   14.7   12.5       200000 (25000, 0.8 GB) 290   261    250
// (4 heads of 64 are the same by workgroups and bytes.)  One part would still be the
// faster from 512 to 1024 workgroups, by 2.3 us at most.
constexpr unsigned kFewReads = 512;
constexpr int64_t kPastCaches = int64_t{32} << 20;

struct ScaledReadArgs {
  PagedRel rel;
  const uint8_t* codes[2];   // key, value
  const float* scales[2];
  int64_t slot[2], head[2];
  void* out[2];
  int heads, D;
  unsigned block;
  int64_t rows;
};

// A thread per 8 values of a row and kRead rows' parts at once, keys and values alike;
// consecutive threads hold a row's consecutive parts.
// Bound: memory (codes read, twice as many bytes written; those 64000 rows 5.8 TB/s
// where floors are counted at 6.2).
template <int DT, int CODE, int kRead, bool PAST>
__global__ __launch_bounds__(256) void read_kernel(ScaledReadArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  const PagedRel& r = a.rel;
  const unsigned per_head = static_cast<unsigned>(a.D / 8), parts = a.heads * per_head;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (256 * kRead) + threadIdx.x;
  int64_t row[kRead];
  unsigned part[kRead];
  int slot[kRead];
#pragma unroll
  for (int u = 0; u < kRead; ++u) {
    const int64_t i = first + 256 * u;
    slot[u] = -1;
    row[u] = a.rows;
    if (i >= a.rows * parts) continue;
    row[u] = i / parts;
    part[u] = static_cast<unsigned>(i - row[u] * parts);
    // (Rows are fewer than 2^31.)
    const int b = static_cast<unsigned>(row[u]) / static_cast<unsigned>(r.queries);
    const int pos = paged_length(r, b) - r.queries + (static_cast<int>(row[u]) - b * r.queries);
    if (pos >= 0) slot[u] = paged_slot(r, r.table + b * r.seq_stride, pos);
  }
  u32x2 w[kRead][2];
  float s[kRead][2];
#pragma unroll
  for (int u = 0; u < kRead; ++u) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      w[u][which] = u32x2{0u, 0u};
      s[u][which] = 0.f;
      if (slot[u] < 0) continue;
      const int h = part[u] / per_head, d = part[u] % per_head * 8;
      w[u][which] = *reinterpret_cast<const u32x2*>(a.codes[which] + slot[u] * a.slot[which] +
                                                    h * a.head[which] + d);
      s[u][which] = a.scales[which][static_cast<int64_t>(slot[u] / a.block) * a.heads + h];
    }
  }
#pragma unroll
  for (int u = 0; u < kRead; ++u) {
    if (row[u] >= a.rows) continue;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float f[8];
      widen8<CODE>(w[u][which], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= s[u][which];
      T* to = static_cast<T*>(a.out[which]) + (row[u] * parts + part[u]) * 8;
      if constexpr (PAST && DT != TGX_DTYPE_F32) {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = DT == TGX_DTYPE_BF16 ? pack_bf16x2(f[2 * i], f[2 * i + 1])
                                      : pack_f16x2(f[2 * i], f[2 * i + 1]);
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to));
      } else {
        V::store(to, f);
      }
    }
  }
}

// f(std::integral_constant<int, dtype>, std::integral_constant<int, code>)
template <typename F>
int with_types(int dtype, int code, F&& f) {
  auto by_code = [&](auto dt) {
    return code == TGX_CODE_E4M3 ? f(dt, std::integral_constant<int, TGX_CODE_E4M3>{})
                                 : f(dt, std::integral_constant<int, TGX_CODE_INT8>{});
  };
  if (dtype == TGX_DTYPE_BF16) return by_code(std::integral_constant<int, TGX_DTYPE_BF16>{});
  if (dtype == TGX_DTYPE_F16) return by_code(std::integral_constant<int, TGX_DTYPE_F16>{});
  return by_code(std::integral_constant<int, TGX_DTYPE_F32>{});
}

int check_scaled(const tgx_paged* p, int heads, int D, int dtype, int code, int block) {
  if (int st = check_paged(p)) return st;
  TGX_REQUIRE(p->table_heads == 1, "one page table per sequence");
  TGX_REQUIRE(heads >= 1 && dtype_bytes(dtype) != 0 && known_code(code), 
              "bad heads, dtype or code");
  if (D < 8 || D > 512 || D % 8) {
    set_error("rows of %d values: caches in 8 bits take multiples of 8 up to 512", D);
    return TGX_UNSUPPORTED;
  }
  TGX_REQUIRE(block >= 1 && p->page_size % block == 0,
              "pages of %d slots are no whole blocks of %d", p->page_size, block);
  return TGX_OK;
}

bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_paged_append_scaled(const tgx_paged* p, void* key_codes_dev,
                                       float* key_scales_dev, const void* key_dev,
                                       void* value_codes_dev, float* value_scales_dev,
                                       const void* value_dev, const int64_t* strides,
                                       float* page_sums_dev, int heads, int D, int dtype, int code,
                                       int block, void* stream) {
  if (int st = check_scaled(p, heads, D, dtype, code, block)) return st;
  if (p->n_seqs == 0 || p->num_pages == 0 || p->pages_per_seq == 0) return TGX_OK;
  TGX_REQUIRE(key_codes_dev && key_scales_dev && key_dev && value_codes_dev && value_scales_dev &&
                  value_dev && strides,
              "null operand");
  TGX_REQUIRE(on(key_codes_dev, 8) && on(value_codes_dev, 8) && on(key_dev, 16) &&
                  on(value_dev, 16),
              "codes must start on 8 bytes and rows on 16");
  const int vec = 16 / dtype_bytes(dtype);
  for (int i = 0; i < 8; ++i)
    TGX_REQUIRE(strides[i] % (i % 4 < 2 ? 8 : vec) == 0, "stride %lld does not keep rows aligned",
                static_cast<long long>(strides[i]));
  const int touched = static_cast<int>(
      std::min<int64_t>(p->pages_per_seq, (int64_t{p->queries} - 1) / p->page_size + 2));
  const int64_t blocks = p->n_seqs * touched;
  const int groups = p->page_size == block ? (heads + 1) / 2 : heads;
  if (blocks > kMaxBlocks256 / groups - 8) {
    set_error("append: too many sequences, pages and heads for one launch");
    return TGX_UNSUPPORTED;
  }
  ScaledAppendArgs a{paged_rel(*p),
                     static_cast<uint8_t*>(key_codes_dev),
                     static_cast<uint8_t*>(value_codes_dev),
                     key_scales_dev,
                     value_scales_dev,
                     key_dev,
                     value_dev,
                     strides[0],
                     strides[1],
                     strides[4],
                     strides[5],
                     strides[2],
                     strides[3],
                     strides[6],
                     strides[7],
                     page_sums_dev,
                     heads,
                     D,
                     block,
                     touched};
  hipStream_t s = as_stream(stream);
  TGX_PROFILE("append_scaled", s);
  with_types(dtype, code, [&](auto dt, auto cd) {
    constexpr int DT = decltype(dt)::value, CODE = decltype(cd)::value;
    const dim3 grid(static_cast<uint32_t>(ceil_div(blocks, 8) * 8 * groups));
    if (D <= 64) append_scaled_kernel<DT, 8, CODE><<<grid, dim3(256), 0, s>>>(a);
    else if (D <= 128) append_scaled_kernel<DT, 16, CODE><<<grid, dim3(256), 0, s>>>(a);
    else append_scaled_kernel<DT, 64, CODE><<<grid, dim3(256), 0, s>>>(a);
    return 0;
  });
  TGX_LAUNCHED("append_scaled");
  return TGX_OK;
}

extern "C" int tgx_paged_read(const tgx_paged* p, const void* key_codes_dev,
                              const float* key_scales_dev, const void* value_codes_dev,
                              const float* value_scales_dev, const int64_t* strides, void* key_dev,
                              void* value_dev, int heads, int D, int dtype, int code, int block,
                              void* stream) {
  if (int st = check_scaled(p, heads, D, dtype, code, block)) return st;
  if (p->n_seqs == 0) return TGX_OK;
  TGX_REQUIRE(key_dev && value_dev && strides, "null operand");
  TGX_REQUIRE(p->num_pages == 0 ||
                  (key_codes_dev && key_scales_dev && value_codes_dev && value_scales_dev),
              "null cache");
  TGX_REQUIRE(on(key_codes_dev, 8) && on(value_codes_dev, 8) && on(key_dev, 16) &&
                  on(value_dev, 16),
              "codes must start on 8 bytes and rows on 16");
  for (int i = 0; i < 4; ++i)
    TGX_REQUIRE(strides[i] % 8 == 0, "stride %lld does not keep codes on 8 bytes",
                static_cast<long long>(strides[i]));
  ScaledReadArgs a{paged_rel(*p),
                   {static_cast<const uint8_t*>(key_codes_dev),
                    static_cast<const uint8_t*>(value_codes_dev)},
                   {key_scales_dev, value_scales_dev},
                   {strides[0], strides[2]},
                   {strides[1], strides[3]},
                   {key_dev, value_dev},
                   heads,
                   D,
                   static_cast<unsigned>(block),
                   p->n_seqs * p->queries};
  // Without pages there is no slot to read, whatever the lengths say.
  if (p->num_pages == 0) a.rel.pages_per_seq = 0;
  const int64_t parts = a.rows * heads * (D / 8);
  if (ceil_div(parts, 1024) > kMaxBlocks256) {
    set_error("read: too many rows for one launch");
    return TGX_UNSUPPORTED;
  }
  hipStream_t s = as_stream(stream);
  TGX_PROFILE("paged_read", s);
  with_types(dtype, code, [&](auto dt, auto cd) {
    constexpr int DT = decltype(dt)::value, CODE = decltype(cd)::value;
    const dim3 one(static_cast<uint32_t>(std::min(ceil_div(parts, 256), kMaxBlocks256)));
    const dim3 four(static_cast<uint32_t>(ceil_div(parts, 1024)));
    const bool past = 16 * parts * dtype_bytes(dtype) > kPastCaches;
    if (four.x < kFewReads) read_kernel<DT, CODE, 1, false><<<one, dim3(256), 0, s>>>(a);
    else if (past) read_kernel<DT, CODE, 4, true><<<four, dim3(256), 0, s>>>(a);
    else read_kernel<DT, CODE, 4, false><<<four, dim3(256), 0, s>>>(a);
    return 0;
  });
  TGX_LAUNCHED("paged_read");
  return TGX_OK;
}
