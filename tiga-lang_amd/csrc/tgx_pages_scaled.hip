// Upkeep of a paged cache held in 8 bits (Graph.append on tiga.BlockScaled) and
// reading it back (Graph.read).
//
// append: the newest tokens' rows x of a block of `block` slots, for each head, with
// M the largest code:
//
//   s' = the smallest power of two >= 2^-126 with max |x| <= M s'
//   s  = max(s', the scale of the block's older tokens), s' where there are none
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

// One workgroup per (sequence, touched page, head), a wave per block of the page in
// turn: LPR lanes hold a row, 8 values each, and 64 / LPR rows are taken at a time.
// A block's new rows are read twice, the second time from the caches.
// Bound: memory for prompts (16-bit rows read, codes written), latency for a single
// token.
template <int DT, int LPR, int CODE>
__global__ __launch_bounds__(256) void append_scaled_kernel(ScaledAppendArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  constexpr int RPI = 64 / LPR;
  __shared__ float part[4 * RPI][LPR * 8];
  const PagedRel& r = a.rel;
  const int h = blockIdx.x % a.heads;
  const int item = blockIdx.x / a.heads;
  const int b = item / a.touched;
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
  const int sub = lane / LPR, d = lane % LPR * 8;
  const bool has = d < a.D;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.f;

  auto cache = [&](uint8_t* codes, int64_t c_slot, int64_t c_head, float* scales, const void* rows,
                   int64_t x_row, int64_t x_head, bool keys) {
    uint8_t* cb = codes + slot0 * c_slot + h * c_head + d;
    const T* xb = static_cast<const T*>(rows) + row0 * x_row + h * x_head + d;
    const int64_t scale0 = slot0 / a.block * a.heads + h;
    const int first = keys && a.sums ? 0 : old / a.block;
    for (int j = first + wave; j * a.block < held; j += 4) {
      const int s0 = j * a.block, s1 = min(s0 + a.block, held);
      const int from = min(max(old, s0), s1);        // the block's first new slot
      float* at = scales + scale0 + static_cast<int64_t>(j) * a.heads;
      float scale = from > s0 ? *at : 0.f;
      const float before = scale;
      if (from < s1) {
        uint32_t top = 0;
        for (int s = from + sub; s < s1; s += RPI) {
          float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (has) V::unpack(V::load(xb + s * x_row), f);
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
        }
        const float need = block_scale<CODE>(wave_largest(top));
        // (Either one's NaN stays.)
        scale = from == s0 || !(need <= scale) ? (scale != scale ? scale : need) : scale;
        if (lane == 0) *at = scale;
      }
      const bool lost = scale != scale;
      const bool again = from > s0 && from < s1 && scale != before && !lost;
      const float ratio = again ? before / scale : 1.f;
      for (int s = (keys && a.sums) || again ? s0 + sub : from + sub; s < s1; s += RPI) {
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        u32x2 w = {0u, 0u};
        if (has) {
          if (s < from) {
            w = *reinterpret_cast<const u32x2*>(cb + s * c_slot);
            if (again) {
              widen8<CODE>(w, f);
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] *= ratio;
              w = encode8<CODE>(f);
            }
          } else if (!lost) {
            V::unpack(V::load(xb + s * x_row), f);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = f[i] / scale;
            w = encode8<CODE>(f);
          }
          if (s >= from || again) *reinterpret_cast<u32x2*>(cb + s * c_slot) = w;
        }
        if (keys && a.sums) {
          widen8<CODE>(w, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] += f[i] * scale;
        }
      }
    }
  };
  cache(a.kc, a.kc_slot, a.kc_head, a.ks, a.k, a.k_row, a.k_head, true);
  cache(a.vc, a.vc_slot, a.vc_head, a.vs, a.v, a.v_row, a.v_head, false);
  if (!a.sums) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[wave * RPI + sub][d + i] = sum[i];
  __syncthreads();
  for (int c = threadIdx.x; c < a.D; c += 256) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 4 * RPI; ++w) total += part[w][c];
    a.sums[(static_cast<int64_t>(id) * a.heads + h) * a.D + c] = total;
  }
}

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

// A thread per 8 values of a row; a row's chunks are consecutive threads.
// Bound: memory (codes read, twice as many bytes written).
template <int DT, int CODE>
__global__ __launch_bounds__(256) void read_kernel(ScaledReadArgs a) {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  const PagedRel& r = a.rel;
  const unsigned chunks = a.heads * static_cast<unsigned>(a.D / 8);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int b = static_cast<int>(row / r.queries);
    const int pos = paged_length(r, b) - r.queries + static_cast<int>(row % r.queries);
    const int slot = pos < 0 ? -1 : paged_slot(r, r.table + b * r.seq_stride, pos);
    for (unsigned c = threadIdx.x; c < chunks; c += 256) {
      const int h = c / (a.D / 8), d = c % (a.D / 8) * 8;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (slot >= 0) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(
              a.codes[which] + slot * a.slot[which] + h * a.head[which] + d);
          const float s = a.scales[which][static_cast<int64_t>(slot / a.block) * a.heads + h];
          widen8<CODE>(w, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= s;
        }
        V::store(static_cast<T*>(a.out[which]) + (row * a.heads + h) * a.D + d, f);
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
  TGX_REQUIRE(heads >= 1 && dtype_bytes(dtype) != 0 && known_code(code), "bad heads, dtype or code");
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
  if (blocks > kMaxBlocks256 / heads) {
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
    const dim3 grid(static_cast<uint32_t>(blocks * heads));
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
  hipStream_t s = as_stream(stream);
  TGX_PROFILE("paged_read", s);
  with_types(dtype, code, [&](auto dt, auto cd) {
    const int64_t grid = std::min<int64_t>(a.rows, 1 << 20);
    read_kernel<decltype(dt)::value, decltype(cd)::value>
        <<<dim3(static_cast<uint32_t>(grid)), dim3(256), 0, s>>>(a);
    return 0;
  });
  TGX_LAUNCHED("paged_read");
  return TGX_OK;
}
