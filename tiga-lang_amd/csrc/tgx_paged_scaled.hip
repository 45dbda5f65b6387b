// Attention over a paged relation whose cache is held in 8 bits (see
// tgx_paged_attn.h for the formula and the split of the work): each key and value
// row is D codes, with a scale for a block of slots and head.
//
// Bound: half the bytes of a 16-bit cache at the same operations, so memory
// again, with twice the keys a second to convert and weigh.
#include "tgx_paged_attn.h"

namespace tgx {
namespace {

// Up to 16 queries, as paged_tile_kernel: a wave runs through every fourth step of
// K8 keys by itself.  K's codes come 16 a lane, whose halves are two fragments;
// V's become bf16 on their way to the wave's LDS rows.  bf16 holds any code, and a
// weight times a value's scale for any scale, which fp16 would not: so weights
// and values are multiplied in bf16 (two parts a weight) for fp16 queries too.
//
// A workgroup holds four adjacent key heads (two, or one, where they do not divide
// so), a wave each, so that it reads whole stretches of a cache's slots: 4 sequences of
// 100k-131k tokens, 8 x 4 heads of 128 in int8, took 222 us with one head a
// workgroup, 197 with two, 184 with four; 64 sequences of 100-4000 95, 85 and 70 us.
// What is left is the order of the reads: the loads alone, with nothing computed, take
// 177 us.  64 keys a step keep as many bytes in flight at D = 128 as 32 of a 16-bit
// cache (and measured as 32 do); narrower heads would not fit three and four
// workgroups a CU with them.
template <int D>
constexpr int kKeys8 = D == 128 ? 64 : 32;
template <typename T, int D, int CODE, bool WIN>
__global__ __launch_bounds__(256, (D == 128 ? 2 : D == 64 ? 3 : 4)) void paged_tile8_kernel(
    PagedArgs a) {
  using VT = __bf16;
  constexpr int K8 = kKeys8<D>, KT = K8 / 16, PART = 32, PT = PART / 16, ROW = kRow<D>;
  constexpr int BYTES = D == 32 ? 8 : 16, NR = D == 128 ? 2 : 1;   // a lane's part, parts
  using Raw = std::conditional_t<D == 32, u32x2, u32x4>;
  constexpr size_t kStage = sizeof(VT) * 4 * PART * ROW;
  constexpr size_t kWeights = sizeof(float) * 4 * PART * 16;
  constexpr size_t kBytes = kStage + kWeights + sizeof(float) * 4 * 2 * K8;
  __shared__ __align__(16) char smem[kBytes > kJoinBytes<D> ? kBytes : kJoinBytes<D>];
  const PagedRel& r = a.rel;
  const unsigned all_heads = r.heads * a.heads;
  const int rows = r.queries * a.group;
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const Wave wv(a, wave);
  const Piece p = find_piece<WIN>(a, wv.x);
  if (p.seq < 0) return;
  const int th = wv.th, kh = wv.kh, head = wv.head, parts = wv.parts;
  if (a.meta && p.index == 0 && head == 0 && threadIdx.x == 0)
    a.meta[p.seq] = make_int2(wv.x, p.count);

  const int g = lane >> 4, lr = lane & 15;
  const Query<T, D, WIN, D != 32> q(a, p, th, kh, lr, rows, g);
  // What the oldest and the newest of the queries see, and the piece's end.
  const Sight<WIN> oldest(a, p.length - (r.queries - 1)), newest(a, p.length);
  const int high = WIN ? p.length : min(p.length, p.tile1 * kTile);
  const uint8_t* kb = static_cast<const uint8_t*>(a.k) + th * a.ks_table + kh * a.ks_head +
                      BYTES * g;
  const uint8_t* vb = static_cast<const uint8_t*>(a.v) + th * a.vs_table + kh * a.vs_head +
                      BYTES * g;
  const int32_t* table = r.table + p.seq * r.seq_stride + th * r.head_stride;
  // The wave's staged V, its weights where they are taken key by key, and its
  // keys' scales.
  VT* stage = reinterpret_cast<VT*>(smem) + wave * PART * ROW;
  float* weights = reinterpret_cast<float*>(smem + kStage) + wave * PART * 16;
  float* scales = reinterpret_cast<float*>(smem + kStage + kWeights) + wave * 2 * K8;

  const int first = p.tile0 * (kTile / K8) + wv.part;
  constexpr int PER = kTile / K8;
  const int last = WIN ? min(p.tile1 * PER, (high + K8 - 1) / K8 - p.gap.skip * PER)
                       : (high + K8 - 1) / K8;
  auto start = [&](int step) { return (WIN ? p.at(step, PER) : step) * K8; };
  auto page_id = [&](int step) {
    const int pos = min(start(step) + lane % K8, r.pages_per_seq * r.page_size - 1);
    return table[static_cast<unsigned>(pos) / static_cast<unsigned>(r.page_size)];
  };
  auto slot_of = [&](int step, int id) {
    const unsigned pos = start(step) + lane % K8;
    const bool there = static_cast<int>(pos) < high &&
                       (!WIN || (step < last && (static_cast<int>(pos) >= oldest.from ||
                                                 static_cast<int>(pos) < oldest.sinks))) &&
                       static_cast<unsigned>(id) < static_cast<unsigned>(r.num_pages);
    return there ? id * r.page_size + static_cast<int>(pos % static_cast<unsigned>(r.page_size))
                 : -1;
  };
  // (A key that is not there loads slot 0, and is masked.)
  auto load = [&](Raw(&f)[KT][NR], const uint8_t* base, int64_t stride, int slot) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int s = max(__shfl(slot, 16 * kt + lr, 64), 0);
      const uint8_t* row = base + s * stride;
#pragma unroll
      for (int c = 0; c < NR; ++c) f[kt][c] = *reinterpret_cast<const Raw*>(row + 64 * c);
    }
  };
  auto scale_of = [&](const float* by, int slot) {
    const int64_t at = static_cast<int64_t>(static_cast<unsigned>(max(slot, 0)) / a.block);
    return by[at * all_heads + head];
  };

  float m = kNegInf, l = 0.f;
  f32x4 o[1][D / 16];
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) o[0][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (first < last) {
    Raw kf[KT][NR], vf[KT][NR];
    int slot = slot_of(first, page_id(first));
    load(kf, kb, a.ks_slot, slot);
    load(vf, vb, a.vs_slot, slot);
    float ks = scale_of(a.k_scales, slot), vs = scale_of(a.v_scales, slot);
    int next_id = page_id(first + parts);
    for (int step = first; step < last; step += parts) {
      const int next = slot_of(step + parts, next_id);
      next_id = page_id(step + 2 * parts);
      const unsigned long long gone = __ballot(slot < 0);   // bit k: key k is not there
      const float vs_here = slot < 0 ? 0.f : vs;
      if (lane < K8) {
        scales[lane] = slot < 0 ? 0.f : ks * a.scale_log2;
        scales[K8 + lane] = vs_here;
      }
      f32x4 c[1][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) c[0][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          if constexpr (D == 32) {
            c[0][kt] = mfma(__builtin_bit_cast(vec8<T>, code_octet<T, CODE>(kf[kt][i])), q.f[i],
                            c[0][kt]);
          } else {
            const u32x4 w = kf[kt][i];
            c[0][kt] = mfma(__builtin_bit_cast(vec8<T>, code_octet<T, CODE>(u32x2{w[0], w[1]})),
                            q.f[2 * i], c[0][kt]);
            c[0][kt] = mfma(__builtin_bit_cast(vec8<T>, code_octet<T, CODE>(u32x2{w[2], w[3]})),
                            q.f[2 * i + 1], c[0][kt]);
          }
        }
      load(kf, kb, a.ks_slot, next);
      ks = scale_of(a.k_scales, next);

      const int pos = start(step);
      const bool part = !oldest.all(pos, K8, newest);   // some query sees only a part
      __builtin_amdgcn_wave_barrier();
      f32x4 by[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        c[0][kt] *= *reinterpret_cast<const f32x4*>(scales + 16 * kt + 4 * g);
        by[kt] = *reinterpret_cast<const f32x4*>(scales + K8 + 16 * kt + 4 * g);
      }
      weigh<VT, WIN>(c[0], gone || part, gone, pos, q.sees, g, m, l, o[0]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) c[0][kt] *= by[kt];

      // V by 32 keys through the wave's rows; a key that is not there counts as a
      // row of zeros.
      if (gone) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
          if (gone >> (16 * kt + lr) & 1) {
#pragma unroll
            for (int i = 0; i < NR; ++i) vf[kt][i] = Raw{};
          }
      }
#pragma unroll
      for (int half = 0; half < K8 / PART; ++half) {
        // A NaN among the values matters where some query does not see all keys.
        Largest<VT> largest;
        if (half) __builtin_amdgcn_wave_barrier();   // the rows before have been read
#pragma unroll
        for (int k = 0; k < PT; ++k)
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            const Raw raw = vf[half * PT + k][i];
            VT* to = stage + (16 * k + lr) * ROW + 64 * i + BYTES * g;
            const vec8<VT> lo =
                __builtin_bit_cast(vec8<VT>, code_octet<VT, CODE>(u32x2{raw[0], raw[1]}));
            if (CODE != TGX_CODE_INT8 && part) largest.see(lo);
            *reinterpret_cast<vec8<VT>*>(to) = lo;
            if constexpr (D != 32) {
              const vec8<VT> hi =
                  __builtin_bit_cast(vec8<VT>, code_octet<VT, CODE>(u32x2{raw[2], raw[3]}));
              if (CODE != TGX_CODE_INT8 && part) largest.see(hi);
              *reinterpret_cast<vec8<VT>*>(to + 8) = hi;
            }
          }
        const bool odd = part && __any(largest.odd() || !(fabsf(vs_here) < __builtin_huge_valf()));
        if (half == K8 / PART - 1) {
          load(vf, vb, a.vs_slot, next);
          vs = scale_of(a.v_scales, next);
        }
        __builtin_amdgcn_wave_barrier();
        f32x4 w[1][PT];
#pragma unroll
        for (int k = 0; k < PT; ++k) w[0][k] = c[0][half * PT + k];
        if (!odd)
          add_values<VT, D, PT, 1>(stage, w, g, lr, o);
        else
          add_seen_values<VT, D, WIN>(stage, w[0], g, lr, pos + PART * half, q.sees, weights, o[0]);
      }
      slot = next;
    }
  }
  join_heads<T, D>(a, p, wv, rows, smem, m, l, o[0]);
}

template <typename T, int D, int CODE, bool WIN>
int launch_tiles(const PagedArgs& a, const Cut& cut, int held, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.rel.queries) * a.group;
  const int64_t pieces = cut.launched * a.rel.heads * a.heads;
  TGX_PROFILE("paged_scaled_tiles", stream);
  if (held == 16) {
    const int64_t blocks = ceil_div(cut.launched, 8) * 8 * a.rel.heads * a.heads / a.held;
    paged_tile8_kernel<T, D, CODE, WIN>
        <<<dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream>>>(a);
  } else {
    const dim3 grid(static_cast<uint32_t>(ceil_div(pieces, 8) * 8 * ceil_div(rows, held)));
    // (With the bounds of a window always, for half as many kernels.  They take 1 to 6% at
    // D = 128 and up to 4% at 64: 4 sequences of 3000-4000, 8 x 4 heads of 128, 16 new tokens
    // in int8 29.6 us, 27.9 without, 512 in int8 367 and 360, in e4m3 314 and 304.  At 128
    // queries and D = 128 45 registers spill for e4m3 and 53 for int8, 33 and 41 without.)
    const dim3 all(256);
    if (held == 32) paged_block_kernel<T, D, 2, 1, CODE, true><<<grid, all, 0, stream>>>(a);
    else if (held == 64) paged_block_kernel<T, D, 1, 1, CODE, true><<<grid, all, 0, stream>>>(a);
    else paged_block_kernel<T, D, 1, 2, CODE, true><<<grid, all, 0, stream>>>(a);
  }
  TGX_LAUNCHED("paged_scaled_tiles");
  return TGX_OK;
}

template <int DT, int LPK, int CODE>
int launch_rows(const PagedArgs& a, const Cut& cut, hipStream_t stream) {
  const int64_t queries = static_cast<int64_t>(a.rel.heads) * a.heads * a.rel.queries * a.group;
  if (cut.launched > kMaxBlocks256 / queries) {
    set_error("paged attention: too many sequences, heads and queries for one launch");
    return TGX_UNSUPPORTED;
  }
  TGX_PROFILE("paged_scaled_rows", stream);
  paged_rows_kernel<DT, LPK, CODE, true>
      <<<dim3(static_cast<uint32_t>(cut.launched * queries)), dim3(256), 0, stream>>>(a);
  TGX_LAUNCHED("paged_scaled_rows");
  return TGX_OK;
}

template <int DT, int CODE>
int dispatch_rows(const PagedArgs& a, const Cut& cut, hipStream_t stream) {
  if (a.D <= 32) return launch_rows<DT, 4, CODE>(a, cut, stream);
  if (a.D <= 64) return launch_rows<DT, 8, CODE>(a, cut, stream);
  if (a.D <= 128) return launch_rows<DT, 16, CODE>(a, cut, stream);
  if (a.D <= 256) return launch_rows<DT, 32, CODE>(a, cut, stream);
  return launch_rows<DT, 64, CODE>(a, cut, stream);
}

template <typename T, int CODE>
int dispatch_tiles(const PagedArgs& a, const Cut& cut, int held, hipStream_t stream) {
  const bool win = a.window < a.rel.pages_per_seq * a.rel.page_size;
  auto width = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return win ? launch_tiles<T, D, CODE, true>(a, cut, held, stream)
               : launch_tiles<T, D, CODE, false>(a, cut, held, stream);
  };
  if (a.D == 32) return width(std::integral_constant<int, 32>{});
  if (a.D == 64) return width(std::integral_constant<int, 64>{});
  return width(std::integral_constant<int, 128>{});
}

template <int CODE>
int dispatch(const PagedArgs& a, const Cut& cut, int held, int dtype, hipStream_t stream) {
  switch (dtype) {
    case TGX_DTYPE_BF16:
      return held ? dispatch_tiles<__bf16, CODE>(a, cut, held, stream)
                  : dispatch_rows<TGX_DTYPE_BF16, CODE>(a, cut, stream);
    case TGX_DTYPE_F16:
      return held ? dispatch_tiles<_Float16, CODE>(a, cut, held, stream)
                  : dispatch_rows<TGX_DTYPE_F16, CODE>(a, cut, stream);
    default:
      return dispatch_rows<TGX_DTYPE_F32, CODE>(a, cut, stream);
  }
}

}  // namespace

int paged_attn_scaled(const PagedArgs& a, const Cut& cut, int held, int dtype, int code,
                      hipStream_t stream) {
  return code == TGX_CODE_E4M3 ? dispatch<TGX_CODE_E4M3>(a, cut, held, dtype, stream)
                               : dispatch<TGX_CODE_INT8>(a, cut, held, dtype, stream);
}

}  // namespace tgx
