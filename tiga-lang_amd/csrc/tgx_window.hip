// Causal attention of packed sequences that looks back over a window (Graph.cu_seqlens
// and Graph.triangular with window and sinks), forward and backward: with i and j
// positions in one sequence,
//
//   out[i, h, g] = sum_j p_ij v[j, h],   p_i = softmax_j(scale q[i, h, g] . k[j, h])
//
// over the keys j <= i with i - j < window or j < sinks.  `group` query heads share a
// key head; with dP = dO V^T and delta_i = <dO_i, out_i>,
//
//   dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
//
// Rows.  The query heads of a key head are rows of one tile: row r of a (sequence,
// key head) is position r / group, head r % group.  A tile of 128 rows then spans
// 128 / group positions, reads each key once for all of its heads, and sees few more
// than window + sinks keys; and dK and dV of shared heads are sums over rows in
// registers, without atomics.
//
// Tiles.  Keys in tiles of 64 of the sequence; a query tile runs through those that
// a row of it sees (the sinks', then the window's), masked where it does not see all
// of one.  Bound: the matrix units (4 D operations a pair forward and 10 D backward,
// against some 4 D / window bytes a pair); at two waves a SIMD the latency between
// LDS, products and softmax stays.  17k tokens, 4 x 4 heads of 128, bf16, a window of
// 1024: forward 185 us with a backward to come (490 TFLOP/s of what is seen), dK/dV 385
// us (470), dQ 200 us (680 with the scores and dP that it forms again; keeping dS for it
// would move 1.3 GB); a prompt of 32768, 8 x 4 heads: 700 us (785).
//
// Rounding.  Scores, softmax statistics, delta and all sums are fp32; P and dS are
// rounded to the inputs' type to be multiplied (half a step of each, whose errors do
// not add up in one direction; the sum of the weights is of the rounded ones: of the
// others it would take 3% longer for a tenth of the error).  With a backward to come the
// forward also stores what rounding took from the output (`rest`), for delta: without
// it dQ and dK were 1.5 times (window of 2: 2.4 times) as far off as results rounded
// once are, with it 1.45 times, for 3% of a training step.
//
// Keys and rows that a row does not see never reach it, whatever they hold: a masked
// tile that has a NaN or Inf among what it contracts over is multiplied row by row.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "tgx_attn_tiles.h"
#include "tgx_device.h"
#include "tgx_host.h"
#include "tgx_profile.h"

namespace tgx {
namespace {

constexpr int kRows = 128;   // rows of a query tile (4 waves x 32)
constexpr int kKeys = 64;    // keys of a tile, and rows of the dK/dV pass's block
constexpr int kMaxGroup = 128;
// Strides of a token stay below this, so that an offset in a tile fits 32 bits.
constexpr int64_t kMaxTokenStride = int64_t{1} << 24;

// The running maximum m moves when a tile's exceeds it by kRescale (log2 units), and a
// weight is 2^(s - m + kLift): fp16 has no numbers below 2^-24, so its weights fill the
// range up to 2^15, as over pages; and in the backward those are P 2^kLift.  (Unlifted,
// keys of weights below 2^-25 = e^-17.3 of the largest are lost from out and dV.  The
// moves take 1% of a step of 17k tokens.)  dS is as large as the output's gradient
// makes it: below 2^-14 it rounds in steps of 2^-24, so it takes the scaled loss that fp16
// training has.
template <typename T>
struct Weights {
  static constexpr float kRescale = kRescaleLog2, kLift = 0.f, kUnlift = 1.f;
};
template <>
struct Weights<_Float16> {
  static constexpr float kRescale = 1.f, kLift = 14.f, kUnlift = 0x1p-14f;
};

struct Form {
  const int32_t* cu;   // [n_blocks + 1] first tokens of the sequences
  int heads, group;
  int window, sinks;
  uint32_t by_group;   // ceil(2^16 / group): n / group of small n (split_row)
};

template <typename T>
struct WinArgs {
  Form f;
  const int32_t* tasks;
  const T* q;
  const T* k;
  const T* v;
  int64_t q_token, q_head, q_group, k_token, k_head, v_token, v_head;   // elements
  float scale_log2;    // |scale| log2(e); 1 for a scale of 0
  float sign;          // what the queries are multiplied by first: 1, -1 or 0
  T* out;              // [n, heads, group, D]; backward: dO
  T* rest;             // forward: out before rounding less out, or null
  float* lse;          // [n, heads, group]: log2 of the sum of 2^(scores * scale_log2), - kLift
};

// Position and head in the group of the row that lies `r` (< 128) rows behind row
// q0 * group + rem.  Exact: n = rem + r < 256 times the excess (< 1) of by_group over
// 2^16 / group is below 2^16 / group (>= 512), what parts two quotients.
__device__ __forceinline__ void split_row(const Form& f, int q0, int rem, int r, int& pos, int& g) {
  const uint32_t n = static_cast<uint32_t>(rem + r);
  const uint32_t up = (n * f.by_group) >> 16;
  pos = q0 + static_cast<int>(up);
  g = static_cast<int>(n - up * static_cast<uint32_t>(f.group));
}

// (No key is seen from position -1.)
__device__ __forceinline__ bool sees(const Form& f, int q, int key) {
  return key <= q && (q - key < f.window || key < f.sinks);
}
// Whether queries q0 .. q1 see all of the 64 keys from k on, or none of them.
__device__ __forceinline__ bool sees_all(const Form& f, int q0, int q1, int k) {
  return k + kKeys - 1 <= q0 && (q1 - k < f.window || k + kKeys <= f.sinks);
}
__device__ __forceinline__ bool sees_none(const Form& f, int q0, int q1, int k) {
  return k > q1 || (q0 - (k + kKeys - 1) >= f.window && k >= f.sinks);
}

// The key tiles that queries q0 .. q1 run through: tile(v) of v < count.
struct KeyTiles {
  int sinks, skip, count;
  __device__ __forceinline__ KeyTiles(const Form& f, int q0, int q1) {
    const int n = q1 / kKeys + 1, first = max(q0 - f.window + 1, 0) / kKeys;
    sinks = min((f.sinks + kKeys - 1) / kKeys, n);
    skip = max(first - sinks, 0);
    count = n - skip;
  }
  __device__ __forceinline__ int tile(int v) const { return v < sinks ? v : v + skip; }
};

// Whether any of eight 16-bit values is a NaN or Inf.
template <typename T>
__device__ __forceinline__ bool any_odd(const vec8<T>& x) {
  constexpr uint32_t kExponent = std::is_same_v<T, __bf16> ? 0x7F80u : 0x7C00u;
  const u32x4 w = __builtin_bit_cast(u32x4, x);
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    odd |= (w[i] & kExponent) == kExponent || (w[i] >> 16 & kExponent) == kExponent;
  return odd;
}

// A staged tile: 64 rows of D values, filled straight from memory (a wave's load
// writes 1 KB in lane order, so rows are not padded) with a row's 16-byte chunk c at
// place c ^ turn(row).  turn() goes in steps of two: what four rows read of two chunks
// (transposed fragments) falls on distinct banks, and so does what sixteen lanes read
// together of fragments (lanes 0-3, 12-15, 20-27 and so on: four rows each of chunk g
// and of g + 1).  With steps that fill the odd places for rows 8-15 a third of dK/dV's
// LDS cycles were conflicts.
typedef __attribute__((address_space(3))) void lds_void;

// BYTES bytes a lane from memory to `to` + BYTES * lane in LDS.  The load has no result
// in registers, and what it writes is read after loads_done() only.  (Of the compiler's
// builtin every read of LDS that follows waits for it at once, also one of the other
// buffer: dQ of 17k tokens 215 us by it.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // (m0 is nobody else's: it is named all the same)
template <int BYTES>
__device__ __forceinline__ void load_lds(const void* from, void* to) {
  static_assert(BYTES == 16 || BYTES == 4, "a lane brings 16 bytes or 4");
  const uint32_t at = uniform(static_cast<int>(reinterpret_cast<uintptr_t>((lds_void*)to)));
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %0, off"
                 ::"v"(from), "s"(at) : "m0", "memory");
  else
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dword %0, off"
                 ::"v"(from), "s"(at) : "m0", "memory");
}
// 16 bytes a lane from `offset` bytes behind `base`, which is the same for all.
__device__ __forceinline__ void load_lds(const void* base, uint32_t offset, void* to) {
  const uint32_t at = uniform(static_cast<int>(reinterpret_cast<uintptr_t>((lds_void*)to)));
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %0, %1"
               ::"v"(offset), "s"(base), "s"(at) : "m0", "memory");
}
#pragma clang diagnostic pop

template <typename T, int D>
struct Tile {
  static constexpr int kRowBytes = 2 * D, kBytes = 64 * kRowBytes;
  static constexpr int kChunks = D / 8, kRowsPerLoad = 64 / kChunks;
  static constexpr int kLoads = 64 / kRowsPerLoad / 4;   // of each of the four waves
  static __device__ __forceinline__ int turn(int row) {
    return row / (128 / D) % (kChunks / 2) * 2;   // (128 / D rows fill all banks)
  }
  // The row of this lane's part of load i, and the first of the eight values it brings.
  static __device__ __forceinline__ int row(int wave, int i) {
    return (wave * kLoads + i) * kRowsPerLoad + lane_id() / kChunks;
  }
  static __device__ __forceinline__ int col(int r) {
    return (lane_id() % kChunks ^ turn(r)) * 8;
  }
  static __device__ __forceinline__ void load(const T* from, char* tile, int wave, int i) {
    load_lds<16>(from, tile + (wave * kLoads + i) * 1024);
  }
  static __device__ __forceinline__ void load(const T* base, uint32_t offset, char* tile,
                                              int wave, int i) {
    load_lds(base, offset, tile + (wave * kLoads + i) * 1024);
  }
  // Where the lane's fragments begin: eight values of row lr (mod 16) from 8 g on, and
  // what the transposing reads take down the columns.  Row r0 of either is a multiple of 16.
  int at, down;
  __device__ __forceinline__ Tile(int g, int lr) {
    at = lr * kRowBytes + ((g % kChunks) ^ turn(lr)) * 16;
    const int r = 4 * g + (lr >> 2);
    down = r * kRowBytes + (((lr & 3) >> 1) ^ turn(r)) * 16 + (lr & 1) * 8;
  }
  // The same in the other of two buffers.
  __device__ __forceinline__ void flip() {
    at ^= kBytes;
    down ^= kBytes;
  }
  // Values 32 kc + 8 g .. of row r0 + lr of the current buffer of `tiles`.  (What is
  // the same in every step is an instruction's own offset, not a register.)
  __device__ __forceinline__ vec8<T> frag(const char* tiles, int r0, int kc) const {
    return *reinterpret_cast<const vec8<T>*>(tiles + r0 * kRowBytes + (at ^ (kc * 64)));
  }
  // Rows r0 + 4 g .. + 3 and r0 + 16 + 4 g .. + 3 of column 16 dt + lr.
  __device__ __forceinline__ vec8<T> column(const char* tiles, int r0, int dt) const {
    const char* p = tiles + r0 * kRowBytes + (down ^ (dt * 32));
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 16 * kRowBytes));
    const u32x2 aw = __builtin_bit_cast(u32x2, a);
    const u32x2 bw = __builtin_bit_cast(u32x2, b);
    return __builtin_bit_cast(vec8<T>, (u32x4{aw[0], aw[1], bw[0], bw[1]}));
  }
  // Four values of a row from column d (a multiple of 4) on.
  static __device__ __forceinline__ vec4<T> four(const char* tile, int r, int d) {
    return *reinterpret_cast<const vec4<T>*>(tile + r * kRowBytes +
                                             ((d / 8 ^ turn(r % 16)) * 16) + d % 8 * 2);
  }
  // Bit 4 dt + e: whether value 16 dt + 4 g + e of row r is a NaN or Inf.
  static __device__ __forceinline__ uint32_t odd_columns(const char* tile, int r, int g) {
    uint32_t found = 0;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const vec4<T> v = four(tile, r, 16 * dt + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = static_cast<float>(v[e]);
        found |= static_cast<uint32_t>(!(__builtin_fabsf(x) < __builtin_huge_valf()))
                 << (4 * dt + e);
      }
    }
    return found;
  }
  // Whether this thread's part of the tile has a NaN or Inf.
  static __device__ __forceinline__ bool odd(const char* tile) {
    bool found = false;
#pragma unroll
    for (int i = 0; i < kBytes / 4096; ++i)
      found |= any_odd<T>(
          *reinterpret_cast<const vec8<T>*>(tile + (threadIdx.x + 256 * i) * 16));
    return found;
  }
};

// Zeros in the place of this thread's NaN and Inf of the tile.
template <typename T, int D>
__device__ __forceinline__ void clear_odd(char* tile) {
  constexpr uint32_t kExponent = std::is_same_v<T, __bf16> ? 0x7F80u : 0x7C00u;
#pragma unroll 1
  for (int i = threadIdx.x * 4; i < Tile<T, D>::kBytes; i += 1024) {
    uint32_t* w = reinterpret_cast<uint32_t*>(tile + i);
    uint32_t x = *w;
    if ((x & kExponent) == kExponent) x &= 0xFFFF0000u;
    if ((x >> 16 & kExponent) == kExponent) x &= 0xFFFFu;
    *w = x;
  }
}

// Key tiles of a head: rows base .. base + 63 of K and V from `k` and `v` (its rows 0) into
// the tiles `ks` and `vs`.  The parts' offsets are the same for every whole tile; rows
// past the sequence are its last one's again, which no row sees.
template <typename T, int D>
struct KeyLoads {
  using TL = Tile<T, D>;
  const T* k;
  const T* v;
  int64_t k_token, v_token;
  int len;
  uint32_t k_off[TL::kLoads], v_off[TL::kLoads];
  __device__ __forceinline__ KeyLoads(const WinArgs<T>& a, int s0, int h, int length, int wave)
      : k(a.k + s0 * a.k_token + h * a.k_head),
        v(a.v + s0 * a.v_token + h * a.v_head),
        k_token(a.k_token),
        v_token(a.v_token),
        len(length) {
#pragma unroll
    for (int i = 0; i < TL::kLoads; ++i) {
      const int r = TL::row(wave, i), c = TL::col(r);
      k_off[i] = static_cast<uint32_t>(r * static_cast<int>(k_token) + c) * sizeof(T);
      v_off[i] = static_cast<uint32_t>(r * static_cast<int>(v_token) + c) * sizeof(T);
    }
  }
  __device__ __forceinline__ void operator()(int base, char* ks, char* vs, int wave) const {
    if (base + kKeys <= len) {
#pragma unroll
      for (int i = 0; i < TL::kLoads; ++i) {
        TL::load(k + base * k_token, k_off[i], ks, wave, i);
        TL::load(v + base * v_token, v_off[i], vs, wave, i);
      }
      return;
    }
#pragma unroll 1
    for (int i = 0; i < TL::kLoads; ++i) {
      const int r = TL::row(wave, i), key = min(base + r, len - 1), c = TL::col(r);
      TL::load(k + key * k_token + c, ks, wave, i);
      TL::load(v + key * v_token + c, vs, wave, i);
    }
  }
};

// Waits for this wave's loads into LDS and joins the workgroup.
__device__ __forceinline__ void loads_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Whether any thread of the workgroup has `mine` (a barrier; `room`: four words of
// LDS that are written once between two barriers of the caller's).
__device__ __forceinline__ bool any_thread(bool mine, int* room) {
  const bool found = __any(mine);
  if (lane_id() == 0) room[threadIdx.x >> 6] = found;
  __syncthreads();
  return room[0] | room[1] | room[2] | room[3];
}

// acc[dt][e] += sum_r w[r][column lr] x[r0 + r][16 dt + 4 g + e] over the 16 rows that the
// column sees (`seen(r)`); w: the wave's 16 x 16 floats of LDS.
template <typename T, int D, typename Seen>
__device__ __forceinline__ void add_seen(const char* x, int r0, const float* w, int g, int lr,
                                         Seen&& seen, f32x4v* acc, int stride) {
#pragma unroll 1
  for (int r = 0; r < 16; ++r) {
    if (!seen(r)) continue;
    const float by = w[r * 16 + lr];
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const vec4<T> v = Tile<T, D>::four(x, r0 + r, 16 * dt + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[dt * stride][e] += by * static_cast<float>(v[e]);
    }
  }
}

// ---------------------------------------------------------------------------
// Forward: a workgroup per tile of 128 rows, a wave per 32 of them, tiles of keys two
// deep in LDS with one barrier each (the prompt of 32768: 782 us with tiles staged
// through registers, 726 so, 700 with parts' offsets formed once), as the dense tiles
// do it: S^T = K Q^T, so that a lane's results are four keys of one row for
// each 16 keys, which is P^T as the B operand of O^T = V^T P^T.

template <typename T, int D>
__global__ __launch_bounds__(256, kFwdWaves<D>) void window_fwd_kernel(WinArgs<T> a) {
  constexpr int KC = D / 32, DT = D / 16;
  using TL = Tile<T, D>;
  __shared__ __align__(1024) char tiles_s[2][2][TL::kBytes];
  auto& ks = tiles_s[0];
  auto& vs = tiles_s[1];
  __shared__ int sh_odd[4];
  const Form& f = a.f;
  const int32_t* task = a.tasks + 4 * static_cast<int64_t>(blockIdx.x);
  const int blk = task[0];
  if (blk < 0) return;   // padding slot of a shorter XCD queue
  const int row0 = task[1], h = task[2];
  const int s0 = f.cu[blk], len = f.cu[blk + 1] - s0;
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, lr = lane & 15;
  const int q0 = row0 / f.group, rem = row0 % f.group;
  auto pos_of = [&](int r) {   // position of a row of the tile, the last one's past it
    int pos, head;
    split_row(f, q0, rem, r, pos, head);
    return min(pos, len - 1);
  };
  const int q1 = pos_of(kRows - 1);
  const int w0 = uniform(pos_of(32 * wave)), w1 = uniform(pos_of(32 * wave + 31));

  // Q^T fragments (B operand): lane holds eight values of row 32 wave + 16 qt + lr.
  vec8<T> qf[2][KC];
  int qpos[2];
  int64_t at[2];   // of the row in out and lse; -1 past the sequence
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    int head;
    split_row(f, q0, rem, 32 * wave + 16 * qt + lr, qpos[qt], head);
    const bool ok = qpos[qt] < len;
    const int64_t token = int64_t{s0} + qpos[qt];
    at[qt] = ok ? (token * f.heads + h) * f.group + head : -1;
    const T* row = a.q + token * a.q_token + h * a.q_head + head * a.q_group;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      qf[qt][kc] = ok ? ld8(row + 32 * kc + 8 * g) : vec8<T>{};
      if (a.sign != 1.f) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          qf[qt][kc][e] = static_cast<T>(static_cast<float>(qf[qt][kc][e]) * a.sign);
      }
    }
    qpos[qt] = min(qpos[qt], len - 1);
  }

  const KeyTiles tiles(f, q0, q1);
  const float sl2 = a.scale_log2;
  float m[2] = {kNegInf, kNegInf};
  f32x4v o[DT][2];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) o[dt][qt] = f32x4v{0.f, 0.f, 0.f, 0.f};
  // The sums of the weights: a row of ones times P^T.
  f32x4v lsum[2] = {f32x4v{0.f, 0.f, 0.f, 0.f}, f32x4v{0.f, 0.f, 0.f, 0.f}};
  vec8<T> ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = static_cast<T>(1.f);

  TL tl(g, lr);
  const KeyLoads<T, D> keys(a, s0, h, len, wave);
  auto load = [&](int v) { keys(tiles.tile(v) * kKeys, ks[v & 1], vs[v & 1], wave); };
  load(0);
  for (int v = 0; v < tiles.count; ++v) {
    loads_done();
    const int buf = v & 1;
    const int kbase = tiles.tile(v) * kKeys;
    if (v + 1 < tiles.count) load(v + 1);
    // (Where some row of the workgroup sees only a part of the tile.)
    bool odd = false;
    if (!sees_all(f, q0, q1, kbase)) odd = any_thread(TL::odd(vs[buf]), sh_odd);

    const bool active = !sees_none(f, w0, w1, kbase);
    f32x4v c[4][2];
    if (active) {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) c[kt][qt] = f32x4v{0.f, 0.f, 0.f, 0.f};
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const vec8<T> kf = tl.frag(ks[0], 16 * kt, kc);
#pragma unroll
          for (int qt = 0; qt < 2; ++qt) c[kt][qt] = mfma(kf, qf[qt][kc], c[kt][qt]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      if (!sees_all(f, w0, w1, kbase)) {
#pragma unroll
        for (int qt = 0; qt < 2; ++qt)
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!sees(f, qpos[qt], kbase + 16 * kt + 4 * g + r)) c[kt][qt][r] = kNegInf;
      }
      float mt[2];
      bool grow = false;
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        float x = kNegInf;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) x = fmaxf(x, c[kt][qt][r]);
        mt[qt] = group4_max(x) * sl2;
        // (The difference: a sum may round away from where m is large.)
        grow |= mt[qt] - m[qt] > Weights<T>::kRescale;
      }
      if (__any(grow)) {
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) {
          const float mn = fmaxf(m[qt], mt[qt]);
          const float alpha = mn == kNegInf ? 1.f : exp2_hw(m[qt] - mn);
          lsum[qt] *= alpha;
          m[qt] = mn;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt][qt] *= alpha;
        }
      }
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        const float mo = m[qt] == kNegInf ? 0.f : m[qt] - Weights<T>::kLift;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) c[kt][qt][r] = exp2_hw(c[kt][qt][r] * sl2 - mo);
      }
      if (!odd) {
        vec8<T> pf[2][2];
#pragma unroll
        for (int qt = 0; qt < 2; ++qt)
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              pf[qt][k2][j] = static_cast<T>(c[2 * k2][qt][j]);
              pf[qt][k2][4 + j] = static_cast<T>(c[2 * k2 + 1][qt][j]);
            }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const vec8<T> vf = tl.column(vs[0], 32 * k2, dt);
#pragma unroll
            for (int qt = 0; qt < 2; ++qt) o[dt][qt] = mfma(vf, pf[qt][k2], o[dt][qt]);
          }
#pragma unroll
          for (int qt = 0; qt < 2; ++qt) lsum[qt] = mfma(ones, pf[qt][k2], lsum[qt]);
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }
    if (odd) {
      // (Uniform: every wave of the workgroup comes here.)  K has been read: its
      // rows hold each wave's weights of 16 keys and 16 rows at a time.
      __syncthreads();
      if (active) {
        float* w = reinterpret_cast<float*>(ks[buf]) + wave * 256;
#pragma unroll
        for (int qt = 0; qt < 2; ++qt)
#pragma unroll
          for (int kt = 0; kt < 4; ++kt) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r = 0; r < 4; ++r) w[(4 * g + r) * 16 + lr] = c[kt][qt][r];
            __builtin_amdgcn_wave_barrier();
            const int key0 = kbase + 16 * kt;
            add_seen<T, D>(
                vs[buf], 16 * kt, w, g, lr, [&](int r) { return sees(f, qpos[qt], key0 + r); },
                &o[0][qt], 2);
            float sum = 0.f;
#pragma unroll 1
            for (int r = 0; r < 16; ++r) sum += w[r * 16 + lr];
            lsum[qt] += sum;
          }
      }
    }
    tl.flip();
  }

#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    if (at[qt] < 0) continue;
    const float l = lsum[qt][0];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* row = a.out + at[qt] * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      vec4<T> w, rest;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = o[dt][qt][r] * inv;
        w[r] = static_cast<T>(x);
        rest[r] = static_cast<T>(x - static_cast<float>(w[r]));
      }
      *reinterpret_cast<vec4<T>*>(row + 16 * dt + 4 * g) = w;
      if (a.rest) *reinterpret_cast<vec4<T>*>(a.rest + at[qt] * D + 16 * dt + 4 * g) = rest;
    }
    // (l is lifted itself.)
    if (g == 0) a.lse[at[qt]] = m[qt] + __log2f(l) - 2.f * Weights<T>::kLift;
  }
}

// ---------------------------------------------------------------------------
// Backward: delta per row; dK/dV, a workgroup per key tile running through the blocks of
// 64 rows that see it; dQ, a workgroup per query tile as the forward.

template <typename T, int D>
__global__ __launch_bounds__(256) void window_delta_kernel(const T* __restrict__ dout,
                                                           const T* __restrict__ out,
                                                           const T* __restrict__ rest,
                                                           float* __restrict__ delta,
                                                           int64_t rows) {
  constexpr int LPR = D / 8;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LPR;
  float s = 0.f;
  if (row < rows) {
    const int64_t off = row * D + threadIdx.x % LPR * 8;
    const vec8<T> x = ld8(dout + off), y = ld8(out + off), z = ld8(rest + off);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      s += static_cast<float>(x[j]) * (static_cast<float>(y[j]) + static_cast<float>(z[j]));
  }
  s = group_sum<LPR>(s);
  if (row < rows && threadIdx.x % LPR == 0) delta[row] = s * Weights<T>::kUnlift;
}

template <typename T>
struct WinBwdArgs {
  WinArgs<T> a;        // out: dO
  const float* delta;  // times kUnlift
  float scale;
  T* dq;               // [n, heads, group, D]
  T* dk;               // [n, heads, D]
  T* dv;
  float* partial;      // [slot, dK and dV (by 1 / kUnlift), 64 keys, D]
};

// dK/dV.  Task: (sequence, first key, head, first block of 64 rows, blocks, slot).  A
// tile with sinks is seen by every later row of its sequence: its rows are cut into
// several tasks, whose sums go to their slots and are joined in order.  Wave w owns keys
// 16 w .. +16; S = Q K^T and dP = dO V^T give P and dS in C layout [row][key], the B
// operand of dV^T = dO^T P and dK^T = Q^T dS.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void window_dkdv_kernel(WinBwdArgs<T> b) {
  constexpr int KC = D / 32, DT = D / 16;
  using TL = Tile<T, D>;
  __shared__ __align__(1024) char tiles_s[2][2][TL::kBytes];
  auto& qs = tiles_s[0];
  auto& dos = tiles_s[1];
  __shared__ __align__(16) float lse_s[2][kKeys], del_s[2][kKeys];
  __shared__ __align__(16) int pos_s[2][kKeys];
  __shared__ float sh_w[4][2][256];   // P and dS of 16 rows and 16 keys, a wave's
  __shared__ int sh_odd[4];
  const WinArgs<T>& a = b.a;
  const Form& f = a.f;
  const int32_t* task = a.tasks + 8 * static_cast<int64_t>(blockIdx.x);
  const int blk = task[0];
  if (blk < 0) return;   // padding slot of a shorter XCD queue
  const int k0 = task[1], h = task[2], block0 = task[3], blocks = task[4], slot = task[5];
  const int s0 = f.cu[blk], len = f.cu[blk + 1] - s0;
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, lr = lane & 15;
  const int key = k0 + 16 * wave + lr;   // this lane's key (B operand column)

  vec8<T> kf[KC], vf[KC];
  {
    const T* krow = a.k + (s0 + key) * a.k_token + h * a.k_head + 8 * g;
    const T* vrow = a.v + (s0 + key) * a.v_token + h * a.v_head + 8 * g;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      kf[kc] = key < len ? ld8(krow + 32 * kc) : vec8<T>{};
      vf[kc] = key < len ? ld8(vrow + 32 * kc) : vec8<T>{};
    }
  }
  const float score_log2 = a.scale_log2 * a.sign;
  f32x4v dkt[DT], dvt[DT];   // dK^T and dV^T [d = 16 dt + 4 g + e][key]
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    dkt[dt] = f32x4v{0.f, 0.f, 0.f, 0.f};
    dvt[dt] = f32x4v{0.f, 0.f, 0.f, 0.f};
  }

  TL tl(g, lr);
  // Where the group divides 64 the parts' offsets are the same for every whole block.
  const bool even = kKeys % f.group == 0 && a.q_token < kMaxTokenStride &&
                    a.q_group < kMaxTokenStride &&
                    int64_t{f.heads} * f.group * D < kMaxTokenStride;
  uint32_t q_off[TL::kLoads], d_off[TL::kLoads];
#pragma unroll
  for (int i = 0; i < TL::kLoads; ++i) {
    const int r = TL::row(wave, i), c = TL::col(r);
    int pos, head;
    split_row(f, 0, 0, r, pos, head);
    q_off[i] = static_cast<uint32_t>(pos * static_cast<int>(a.q_token) +
                                     head * static_cast<int>(a.q_group) + c) * sizeof(T);
    d_off[i] = static_cast<uint32_t>((pos * f.heads * f.group + head) * D + c) * sizeof(T);
  }
  // Rows 64 block .. +63; past the sequence its last one's again, at no position.
  auto load = [&](int block, int buf) {
    const int q0 = block * kKeys / f.group, rem = block * kKeys % f.group;
    if (wave < 2) {
      int pos, head;
      split_row(f, q0, rem, lane, pos, head);
      const int64_t token = s0 + min(pos, len - 1);
      const int64_t at = (token * f.heads + h) * f.group + head;
      if (wave == 0) {
        load_lds<4>(a.lse + at, lse_s[buf]);
        pos_s[buf][lane] = pos < len ? pos : -1;
      } else {
        load_lds<4>(b.delta + at, del_s[buf]);
      }
    }
    if (even && q0 + kKeys / f.group <= len) {
      const T* qb = a.q + (s0 + q0) * a.q_token + h * a.q_head;
      const T* db = a.out + (static_cast<int64_t>(s0 + q0) * f.heads + h) * f.group * D;
#pragma unroll
      for (int i = 0; i < TL::kLoads; ++i) {
        TL::load(qb, q_off[i], qs[buf], wave, i);
        TL::load(db, d_off[i], dos[buf], wave, i);
      }
      return;
    }
#pragma unroll 1
    for (int i = 0; i < TL::kLoads; ++i) {
      const int r = TL::row(wave, i), c = TL::col(r);
      int pos, head;
      split_row(f, q0, rem, r, pos, head);
      const int64_t token = s0 + min(pos, len - 1);
      TL::load(a.q + token * a.q_token + h * a.q_head + head * a.q_group + c, qs[buf], wave, i);
      TL::load(a.out + ((token * f.heads + h) * f.group + head) * D + c, dos[buf], wave, i);
    }
  };
  if (blocks > 0) load(block0, 0);
  for (int step = 0; step < blocks; ++step) {
    const int row0 = (block0 + step) * kKeys, buf = step & 1;
    const int p0 = row0 / f.group, p1 = (row0 + kKeys - 1) / f.group;
    // Some row sees only a part of the tile, or is none.
    const bool part = p1 >= len || !sees_all(f, p0, p1, k0);
    loads_done();
    if (step + 1 < blocks) load(block0 + step + 1, buf ^ 1);
    bool odd = false;
    if (part) odd = any_thread(TL::odd(qs[buf]) || TL::odd(dos[buf]), sh_odd);

    f32x4v sc[4], dp[4];
#pragma unroll
    for (int qt = 0; qt < 4; ++qt) {
      sc[qt] = f32x4v{0.f, 0.f, 0.f, 0.f};
      dp[qt] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) {
        const vec8<T> qa = tl.frag(qs[0], 16 * qt, kc);
        const vec8<T> da = tl.frag(dos[0], 16 * qt, kc);
        sc[qt] = mfma(qa, kf[kc], sc[qt]);
        dp[qt] = mfma(da, vf[kc], dp[qt]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    vec8<T> pb[2], sb[2];
    auto weights = [&](auto masked) {
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) {
        const f32x4v lse = *reinterpret_cast<const f32x4v*>(&lse_s[buf][16 * qt + 4 * g]);
        const f32x4v del = *reinterpret_cast<const f32x4v*>(&del_s[buf][16 * qt + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p = exp2_hw(sc[qt][r] * score_log2 - lse[r]);
          float ds = p * (dp[qt][r] * Weights<T>::kUnlift - del[r]);
          if (decltype(masked)::value && !sees(f, pos_s[buf][16 * qt + 4 * g + r], key))
            p = ds = 0.f;
          pb[qt >> 1][4 * (qt & 1) + r] = static_cast<T>(p);
          sb[qt >> 1][4 * (qt & 1) + r] = static_cast<T>(ds);
        }
      }
    };
    if (part)
      weights(std::true_type{});
    else
      weights(std::false_type{});
    if (!odd) {
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const vec8<T> ot = tl.column(dos[0], 32 * k2, dt);
          const vec8<T> qtv = tl.column(qs[0], 32 * k2, dt);
          dvt[dt] = mfma(ot, pb[k2], dvt[dt]);
          dkt[dt] = mfma(qtv, sb[k2], dkt[dt]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    } else {
      float (*w)[256] = sh_w[wave];
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[0][(4 * g + r) * 16 + lr] = static_cast<float>(pb[qt >> 1][4 * (qt & 1) + r]);
          w[1][(4 * g + r) * 16 + lr] = static_cast<float>(sb[qt >> 1][4 * (qt & 1) + r]);
        }
        __builtin_amdgcn_wave_barrier();
        auto seen = [&](int r) { return sees(f, pos_s[buf][16 * qt + r], key); };
        add_seen<T, D>(dos[buf], 16 * qt, w[0], g, lr, seen, dvt, 1);
        add_seen<T, D>(qs[buf], 16 * qt, w[1], g, lr, seen, dkt, 1);
      }
    }
    tl.flip();
  }
  if (slot >= 0) {
    float* part = b.partial + static_cast<int64_t>(slot) * 2 * kKeys * D + (16 * wave + lr) * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      *reinterpret_cast<f32x4v*>(part + 16 * dt + 4 * g) = dkt[dt];
      *reinterpret_cast<f32x4v*>(part + kKeys * D + 16 * dt + 4 * g) = dvt[dt];
    }
    return;
  }
  if (key >= len) return;
  const int64_t at = (static_cast<int64_t>(s0 + key) * f.heads + h) * D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    vec4<T> wk, wv;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      wk[r] = static_cast<T>(dkt[dt][r] * b.scale);
      wv[r] = static_cast<T>(dvt[dt][r] * Weights<T>::kUnlift);
    }
    *reinterpret_cast<vec4<T>*>(b.dk + at + 16 * dt + 4 * g) = wk;
    *reinterpret_cast<vec4<T>*>(b.dv + at + 16 * dt + 4 * g) = wv;
  }
}

// Joins the slots of a key tile in order: merge (sequence, first key, head, first slot,
// slots), a thread per 4 values of a key's dK or dV.
template <int D>
constexpr int kMergeBlocks = 2 * kKeys * (D / 4) / 256;

template <typename T, int D>
__global__ __launch_bounds__(256) void window_merge_kernel(WinBwdArgs<T> b,
                                                           const int32_t* __restrict__ merges) {
  const int32_t* mt = merges + 8 * static_cast<int64_t>(blockIdx.x / kMergeBlocks<D>);
  const Form& f = b.a.f;
  const int blk = mt[0], k0 = mt[1], h = mt[2], slot0 = mt[3], count = mt[4];
  const int s0 = f.cu[blk], len = f.cu[blk + 1] - s0;
  const int i = (blockIdx.x % kMergeBlocks<D>) * 256 + threadIdx.x;
  const int d = 4 * (i % (D / 4)), key = i / (D / 4) % kKeys, which = i / (kKeys * (D / 4));
  if (k0 + key >= len) return;
  const float* src = b.partial + ((static_cast<int64_t>(slot0) * 2 + which) * kKeys + key) * D + d;
  f32x4v sum = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < count; ++c)
    sum += *reinterpret_cast<const f32x4v*>(src + static_cast<int64_t>(c) * 2 * kKeys * D);
  sum *= which == 0 ? b.scale : Weights<T>::kUnlift;
  vec4<T> w;
#pragma unroll
  for (int r = 0; r < 4; ++r) w[r] = static_cast<T>(sum[r]);
  *reinterpret_cast<vec4<T>*>((which == 0 ? b.dk : b.dv) +
                              (static_cast<int64_t>(s0 + k0 + key) * f.heads + h) * D + d) = w;
}

// dQ: S^T = K Q^T and dP^T = V dO^T give dS^T, the B operand of dQ^T = K^T dS^T.  In a
// masked tile with a NaN or Inf among K, those count as zeros in the last product, and
// the columns where a row sees one are NaN in the end: such a row has a NaN in dS
// already, or (a score of -inf) a weight of 0, which times Inf is one.  (Multiplying row
// by row, as the other kernels do, needs registers that spill here: a spilled
// fragment's reload waits for the tile in flight.)
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void window_dq_kernel(WinBwdArgs<T> b) {
  constexpr int KC = D / 32, DT = D / 16;
  using TL = Tile<T, D>;
  __shared__ __align__(1024) char tiles_s[2][2][TL::kBytes];
  auto& ks = tiles_s[0];
  auto& vs = tiles_s[1];
  __shared__ int sh_odd[4];
  // A thread's: bit 4 dt + r, dqt[dt][.][r] is no number.  (In registers held over the
  // loop they took 1% of a training step.)
  __shared__ uint32_t bad_s[2][256];
  const WinArgs<T>& a = b.a;
  const Form& f = a.f;
  const int32_t* task = a.tasks + 4 * static_cast<int64_t>(blockIdx.x);
  const int blk = task[0];
  if (blk < 0) return;
  const int row0 = task[1], h = task[2];
  const int s0 = f.cu[blk], len = f.cu[blk + 1] - s0;
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, lr = lane & 15;
  const int q0 = row0 / f.group, rem = row0 % f.group;
  auto pos_of = [&](int r) {
    int pos, head;
    split_row(f, q0, rem, r, pos, head);
    return min(pos, len - 1);
  };
  const int q1 = pos_of(kRows - 1);
  const int w0 = uniform(pos_of(32 * wave)), w1 = uniform(pos_of(32 * wave + 31));
  vec8<T> qf[2][KC], df[2][KC];
  float lse2[2], del[2];
  int qpos[2];
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    int head;
    split_row(f, q0, rem, 32 * wave + 16 * qt + lr, qpos[qt], head);
    const bool ok = qpos[qt] < len;
    const int64_t token = s0 + qpos[qt];
    const int64_t at = (token * f.heads + h) * f.group + head;
    const T* row = a.q + token * a.q_token + h * a.q_head + head * a.q_group;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      qf[qt][kc] = ok ? ld8(row + 32 * kc + 8 * g) : vec8<T>{};
      df[qt][kc] = ok ? ld8(a.out + at * D + 32 * kc + 8 * g) : vec8<T>{};
    }
    lse2[qt] = ok ? a.lse[at] : __builtin_huge_valf();
    del[qt] = ok ? b.delta[at] : 0.f;
    qpos[qt] = min(qpos[qt], len - 1);
  }
  f32x4v dqt[DT][2];   // dQ^T [d = 16 dt + 4 g + r][row]
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) dqt[dt][qt] = f32x4v{0.f, 0.f, 0.f, 0.f};
  bad_s[0][threadIdx.x] = bad_s[1][threadIdx.x] = 0u;
  const KeyTiles tiles(f, q0, q1);
  TL tl(g, lr);
  const float score_log2 = a.scale_log2 * a.sign;
  const KeyLoads<T, D> keys(a, s0, h, len, wave);
  auto load = [&](int v) { keys(tiles.tile(v) * kKeys, ks[v & 1], vs[v & 1], wave); };
  load(0);
  for (int v = 0; v < tiles.count; ++v) {
    const int kbase = tiles.tile(v) * kKeys, buf = v & 1;
    loads_done();
    if (v + 1 < tiles.count) load(v + 1);
    bool odd = false;
    if (!sees_all(f, q0, q1, kbase)) odd = any_thread(TL::odd(ks[buf]), sh_odd);
    const bool active = !sees_none(f, w0, w1, kbase);
    const bool part = !sees_all(f, w0, w1, kbase);
    vec8<T> sb[2][2];
    if (active) {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        f32x4v sc[2], dp[2];
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) {
          sc[qt] = f32x4v{0.f, 0.f, 0.f, 0.f};
          dp[qt] = f32x4v{0.f, 0.f, 0.f, 0.f};
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          const vec8<T> ka = tl.frag(ks[0], 16 * kt, kc);
          const vec8<T> va = tl.frag(vs[0], 16 * kt, kc);
#pragma unroll
          for (int qt = 0; qt < 2; ++qt) {
            sc[qt] = mfma(ka, qf[qt][kc], sc[qt]);
            dp[qt] = mfma(va, df[qt][kc], dp[qt]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
        auto weights = [&](auto masked) {
#pragma unroll
          for (int qt = 0; qt < 2; ++qt) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float p = exp2_hw(sc[qt][r] * score_log2 - lse2[qt]);
              float ds = p * (dp[qt][r] * Weights<T>::kUnlift - del[qt]);
              if (decltype(masked)::value && !sees(f, qpos[qt], kbase + 16 * kt + 4 * g + r))
                ds = 0.f;
              sb[qt][kt >> 1][4 * (kt & 1) + r] = static_cast<T>(ds);
            }
          }
        };
        if (part)
          weights(std::true_type{});
        else
          weights(std::false_type{});
        // (Fragments read ahead past this would not fit the registers at D = 128.)
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (odd) {   // (of the whole workgroup)
      if (active) {
#pragma unroll 1
        for (int r = 0; r < kKeys; ++r) {
          const uint32_t found = Tile<T, D>::odd_columns(ks[buf], r, g);
#pragma unroll
          for (int qt = 0; qt < 2; ++qt)
            if (sees(f, qpos[qt], kbase + r)) bad_s[qt][threadIdx.x] |= found;
        }
      }
      __syncthreads();
      clear_odd<T, D>(ks[buf]);
      __syncthreads();
    }
    if (active) {
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const vec8<T> kta = tl.column(ks[0], 32 * k2, dt);
#pragma unroll
          for (int qt = 0; qt < 2; ++qt) dqt[dt][qt] = mfma(kta, sb[qt][k2], dqt[dt][qt]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    tl.flip();
  }
  // (Where a row goes is found again, not kept in registers over the loop.)
  int again = q0;
  asm volatile("" : "+s"(again));
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    int pos, head;
    split_row(f, again, rem, 32 * wave + 16 * qt + lr, pos, head);
    if (pos >= len) continue;
    T* row = b.dq + ((static_cast<int64_t>(s0 + pos) * f.heads + h) * f.group + head) * D;
    const uint32_t bad = bad_s[qt][threadIdx.x];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      vec4<T> w;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        w[r] = static_cast<T>(bad >> (4 * dt + r) & 1 ? __builtin_nanf("")
                                                      : dqt[dt][qt][r] * b.scale);
      *reinterpret_cast<vec4<T>*>(row + 16 * dt + 4 * g) = w;
    }
  }
}

// ---------------------------------------------------------------------------
// Launches

struct WinShape {
  int64_t n;
  int heads, group, D, dtype;
};

int check_shape(const WinShape& s, const int64_t* strides, int window, int sinks) {
  if (s.D != 32 && s.D != 64 && s.D != 128) {
    set_error("windowed attention tiles support head widths 32, 64 and 128 (got %d)", s.D);
    return TGX_UNSUPPORTED;
  }
  if (s.dtype != TGX_DTYPE_BF16 && s.dtype != TGX_DTYPE_F16) {
    set_error("windowed attention tiles support bf16 and fp16 (dtype code %d)", s.dtype);
    return TGX_UNSUPPORTED;
  }
  TGX_REQUIRE(s.n >= 0 && s.heads >= 1 && s.group >= 1 && s.group <= kMaxGroup,
              "bad sizes: n %lld, heads %d, group %d", static_cast<long long>(s.n), s.heads,
              s.group);
  TGX_REQUIRE(window >= 1 && sinks >= 0, "window must be positive and sinks not negative");
  TGX_REQUIRE(strides != nullptr, "null strides");
  TGX_REQUIRE(s.n * s.group < (int64_t{1} << 31) - 4 * kRows,
              "rows of a key head must be fewer than 2^31");
  for (int i = 0; i < 7; ++i)
    TGX_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0,
                "stride %lld does not keep rows on 16 bytes", static_cast<long long>(strides[i]));
  if (strides[3] >= kMaxTokenStride || strides[5] >= kMaxTokenStride) {
    set_error("windowed attention tiles need token strides of k and v below %lld elements",
              static_cast<long long>(kMaxTokenStride));
    return TGX_UNSUPPORTED;
  }
  return TGX_OK;
}

template <typename T>
WinArgs<T> make_args(const WinShape& s, const int32_t* cu, const void* q, const void* k,
                     const void* v, const int64_t* st, float scale, int window, int sinks) {
  WinArgs<T> a{};
  // No sequence is longer than all tokens: bounds past that hide nothing, and kernels
  // add a tile to these numbers.
  const int most = static_cast<int>(s.n);
  a.f = Form{cu, s.heads, s.group, std::min(window, most), std::min(sinks, most),
             static_cast<uint32_t>((65536 + s.group - 1) / s.group)};
  a.q = static_cast<const T*>(q);
  a.k = static_cast<const T*>(k);
  a.v = static_cast<const T*>(v);
  a.q_token = st[0], a.q_head = st[1], a.q_group = st[2];
  a.k_token = st[3], a.k_head = st[4], a.v_token = st[5], a.v_head = st[6];
  // The largest score is the largest product where the factor is positive.
  a.sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
  a.scale_log2 = scale == 0.f ? 1.f : __builtin_fabsf(scale) * kLog2e;
  return a;
}

// f(T{}, std::integral_constant<int, D>) for the types and widths that check_shape admits.
template <typename F>
int with_tile(const WinShape& s, F&& f) {
  auto width = [&](auto t) -> int {
    if (s.D == 32) return f(t, std::integral_constant<int, 32>{});
    if (s.D == 64) return f(t, std::integral_constant<int, 64>{});
    return f(t, std::integral_constant<int, 128>{});
  };
  return s.dtype == TGX_DTYPE_BF16 ? width(__bf16{}) : width(_Float16{});
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

size_t delta_bytes(int64_t n, int heads, int group) {
  return align_up(sizeof(float) * n * heads * group);
}

// Blocks of 64 rows that see the key tile at k0 of a sequence of `len` tokens, from
// row block `first` on.
struct RowRange {
  int64_t first, blocks;
};
RowRange rows_seeing(int64_t len, int64_t k0, int group, int64_t window, int64_t sinks) {
  const int64_t first = k0 * group / kKeys;   // (k0 is a multiple of 64)
  const int64_t end = k0 < sinks ? len : std::min(len, k0 + kKeys - 1 + window);
  return {first, ceil_div(end * group, kKeys) - first};
}

// Row blocks of a piece of a key tile that holds sinks, which every later row of its
// sequence sees: a window's rows, so that pieces are as long as other tiles' tasks, and
// at least what leaves kMaxPieces of all the work, four for each workgroup that is
// resident at once.  A tile is cut where it has more than two pieces' blocks, so there
// are at most 1.5 kMaxPieces slots (192 MB at D = 128), however many sinks and
// tokens.  131072 tokens, 8 x 4 heads, a window of 128 and 1024 sinks, a training step:
// pieces of a window's rows alone took 4.3 GB of slots and 18.1 ms, so 0.12 GB and 14.5 ms.
constexpr int64_t kMaxPieces = 4 * 2 * 256;
int64_t blocks_of_a_piece(const int32_t* cu, int n_blocks, int heads, int group, int64_t window,
                          int64_t sinks) {
  int64_t total = 0;
  for (int b = 0; b < n_blocks; ++b) {
    const int64_t len = int64_t{cu[b + 1]} - cu[b];
    for (int64_t k0 = 0; k0 < len; k0 += kKeys)
      total += rows_seeing(len, k0, group, window, sinks).blocks;
  }
  return std::max({ceil_div((window + kKeys - 1) * group, kKeys), int64_t{16},
                   ceil_div(total * heads, kMaxPieces)});
}

// (tgx_window_tasks; may throw.)
int window_tasks(const int32_t* cu_host, int n_blocks, int heads, int group, int window, int sinks,
                 int kind, int32_t* tasks_host, int64_t* n_tasks, int64_t* n_slots) {
  TGX_REQUIRE(cu_host && n_tasks && n_slots && n_blocks >= 0 && heads > 0 && group > 0 &&
                  group <= kMaxGroup && window > 0 && sinks >= 0,
              "bad arguments");
  TGX_REQUIRE(kind >= 0 && kind <= 2, "kind must be 0 (query tiles), 1 (key tiles) or 2 (joins)");
  int64_t tiles = 0;   // (beside them there are 1.5 kMaxPieces tasks at most)
  for (int b = 0; b < n_blocks; ++b) {
    const int64_t len = int64_t{cu_host[b + 1]} - cu_host[b];
    TGX_REQUIRE(len >= 0 && cu_host[b] >= 0, "cu_seqlens must be non-decreasing from 0");
    TGX_REQUIRE(len * group < (int64_t{1} << 31) - 4 * kRows,
                "rows of a key head must be fewer than 2^31");
    tiles += kind == 0 ? ceil_div(len * group, kRows) : ceil_div(len, kKeys);
  }
  // (Before any of them is formed.)
  TGX_REQUIRE(tiles * heads < kMaxBlocks256, "too many tasks");
  const int width = kind == 0 ? 4 : 8;
  struct Task {
    int64_t work;
    int32_t v[8];
  };
  std::vector<Task> tasks, joins;
  int64_t slots = 0;
  const int64_t piece =
      kind == 0 ? 0 : blocks_of_a_piece(cu_host, n_blocks, heads, group, window, sinks);
  for (int b = 0; b < n_blocks; ++b) {
    const int64_t len = int64_t{cu_host[b + 1]} - cu_host[b];
    for (int h = 0; h < heads; ++h) {
      if (kind == 0) {
        for (int64_t r = 0; r < len * group; r += kRows) {
          const int64_t q = r / group;
          tasks.push_back(Task{std::min<int64_t>(q, int64_t{window} + sinks) + kKeys,
                               {b, static_cast<int32_t>(r), h, 0}});
        }
        continue;
      }
      for (int64_t k0 = 0; k0 < len; k0 += kKeys) {
        const RowRange rows = rows_seeing(len, k0, group, window, sinks);
        const int32_t key = static_cast<int32_t>(k0);
        if (rows.blocks <= 2 * piece) {
          tasks.push_back(Task{rows.blocks,
                               {b, key, h, static_cast<int32_t>(rows.first),
                                static_cast<int32_t>(rows.blocks), -1, 0, 0}});
          continue;
        }
        const int64_t count = ceil_div(rows.blocks, piece);
        TGX_REQUIRE(slots + count < (int64_t{1} << 31), "too many pieces");
        joins.push_back(Task{0, {b, key, h, static_cast<int32_t>(slots),
                                 static_cast<int32_t>(count), 0, 0, 0}});
        for (int64_t c = 0; c < count; ++c) {
          const int64_t first = rows.first + c * piece;
          const int64_t n = std::min(piece, rows.first + rows.blocks - first);
          tasks.push_back(Task{n, {b, key, h, static_cast<int32_t>(first),
                                   static_cast<int32_t>(n), static_cast<int32_t>(slots++), 0, 0}});
        }
      }
    }
  }
  *n_slots = slots;
  if (kind == 2) {
    *n_tasks = static_cast<int64_t>(joins.size());
    if (tasks_host)
      for (size_t i = 0; i < joins.size(); ++i)
        std::copy(joins[i].v, joins[i].v + 8, tasks_host + 8 * i);
    return TGX_OK;
  }
  // A share of equal work of the list for each XCD, so that tiles which follow each other
  // (and share most of what they read) run on one L2: workgroup i runs on XCD i % 8.
  int64_t total = 0;
  for (const Task& t : tasks) total += t.work;
  std::vector<std::vector<size_t>> queue(kXcds);
  int64_t done = 0;
  for (size_t i = 0; i < tasks.size(); ++i) {
    queue[std::min<int64_t>(kXcds - 1, done * kXcds / std::max<int64_t>(total, 1))].push_back(i);
    done += tasks[i].work;
  }
  // The largest first: the rounds of workgroups then end evenly.
  size_t longest = 0;
  for (auto& x : queue) {
    std::stable_sort(x.begin(), x.end(),
                     [&](size_t i, size_t j) { return tasks[i].work > tasks[j].work; });
    longest = std::max(longest, x.size());
  }
  const int64_t n = static_cast<int64_t>(longest) * kXcds;
  TGX_REQUIRE(n < kMaxBlocks256, "too many tasks");
  *n_tasks = n;
  if (tasks_host)
    for (size_t i = 0; i < longest; ++i)
      for (int x = 0; x < kXcds; ++x) {
        int32_t* dst = tasks_host + width * (static_cast<int64_t>(i) * kXcds + x);
        if (i < queue[x].size()) {
          std::copy(tasks[queue[x][i]].v, tasks[queue[x][i]].v + width, dst);
        } else {
          std::fill(dst, dst + width, 0);
          dst[0] = -1;
        }
      }
  return TGX_OK;
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_window_tasks(const int32_t* cu_host, int n_blocks, int heads, int group,
                                int window, int sinks, int kind, int32_t* tasks_host,
                                int64_t* n_tasks, int64_t* n_slots) {
  try {
    return window_tasks(cu_host, n_blocks, heads, group, window, sinks, kind, tasks_host, n_tasks,
                        n_slots);
  } catch (const std::bad_alloc&) {
    set_error("host allocation failed");
    return TGX_OUT_OF_MEMORY;
  }
}

extern "C" int tgx_window_attn_fwd(const int32_t* cu_dev, const int32_t* tasks_dev,
                                   int64_t n_tasks, const void* q, const void* k, const void* v,
                                   const int64_t* strides, float scale, int window, int sinks,
                                   void* out, void* rest, float* lse, int64_t n, int heads,
                                   int group, int D, int dtype, void* stream) {
  const WinShape s{n, heads, group, D, dtype};
  if (int st = check_shape(s, strides, window, sinks)) return st;
  TGX_REQUIRE(n_tasks >= 0 && n_tasks < kMaxBlocks256, "bad task count");
  if (n == 0 || n_tasks == 0) return TGX_OK;
  TGX_REQUIRE(cu_dev && tasks_dev && q && k && v && out && lse, "null pointer");
  TGX_REQUIRE(on16(q) && on16(k) && on16(v) && on16(out) && on16(rest),
              "operands must start on 16 bytes");
  hipStream_t hs = as_stream(stream);
  return with_tile(s, [&](auto t, auto d) -> int {
    typedef decltype(t) T;
    WinArgs<T> a = make_args<T>(s, cu_dev, q, k, v, strides, scale, window, sinks);
    a.tasks = tasks_dev;
    a.out = static_cast<T*>(out);
    a.rest = static_cast<T*>(rest);
    a.lse = lse;
    TGX_PROFILE("window_fwd", hs);
    window_fwd_kernel<T, decltype(d)::value>
        <<<dim3(static_cast<uint32_t>(n_tasks)), dim3(256), 0, hs>>>(a);
    TGX_LAUNCHED("window_fwd");
    return TGX_OK;
  });
}

extern "C" int tgx_window_attn_bwd_workspace(int64_t n, int64_t n_slots, int heads, int group,
                                             int D, size_t* bytes) {
  TGX_REQUIRE(bytes && n >= 0 && n_slots >= 0 && heads > 0 && group > 0 && D > 0, "bad arguments");
  *bytes = delta_bytes(n, heads, group) + sizeof(float) * n_slots * 2 * kKeys * D;
  return TGX_OK;
}

extern "C" int tgx_window_attn_bwd(const int32_t* cu_dev, const int32_t* q_tasks_dev,
                                   int64_t n_q_tasks, const int32_t* k_tasks_dev,
                                   int64_t n_k_tasks, const int32_t* joins_dev, int64_t n_joins,
                                   int64_t n_slots, const void* q, const void* k, const void* v,
                                   const int64_t* strides, const void* out, const void* rest,
                                   const float* lse, const void* dout, float scale, int window,
                                   int sinks, void* dq, void* dk, void* dv, int64_t n, int heads,
                                   int group, int D, int dtype, void* workspace_dev,
                                   size_t workspace_bytes, void* stream) {
  const WinShape s{n, heads, group, D, dtype};
  if (int st = check_shape(s, strides, window, sinks)) return st;
  TGX_REQUIRE(n_q_tasks >= 0 && n_q_tasks < kMaxBlocks256 && n_k_tasks >= 0 &&
                  n_k_tasks < kMaxBlocks256 && n_joins >= 0 && n_joins <= kMaxBlocks256 / 16 &&
                  n_slots >= 0,
              "bad task counts");
  if (n == 0 || n_q_tasks == 0) return TGX_OK;
  TGX_REQUIRE(cu_dev && q_tasks_dev && k_tasks_dev && q && k && v && out && rest && lse && dout &&
                  dq && dk && dv && (n_joins == 0 || joins_dev),
              "null pointer");
  TGX_REQUIRE(on16(q) && on16(k) && on16(v) && on16(out) && on16(rest) && on16(dout) && on16(dq) &&
                  on16(dk) && on16(dv),
              "operands must start on 16 bytes");
  size_t need = 0;
  if (int st = tgx_window_attn_bwd_workspace(n, n_slots, heads, group, D, &need)) return st;
  TGX_REQUIRE(workspace_bytes >= need && workspace_dev, "workspace of %zu bytes, needs %zu",
              workspace_bytes, need);
  hipStream_t hs = as_stream(stream);
  return with_tile(s, [&](auto t, auto d) -> int {
    typedef decltype(t) T;
    constexpr int DD = decltype(d)::value;
    float* delta = static_cast<float*>(workspace_dev);
    WinBwdArgs<T> b{};
    b.a = make_args<T>(s, cu_dev, q, k, v, strides, scale, window, sinks);
    b.a.out = const_cast<T*>(static_cast<const T*>(dout));
    b.a.lse = const_cast<float*>(lse);
    b.delta = delta;
    b.scale = scale;
    b.dq = static_cast<T*>(dq);
    b.dk = static_cast<T*>(dk);
    b.dv = static_cast<T*>(dv);
    b.partial = reinterpret_cast<float*>(static_cast<char*>(workspace_dev) +
                                         delta_bytes(n, heads, group));
    {
      const int64_t rows = n * heads * group, blocks = ceil_div(rows * (DD / 8), 256);
      TGX_REQUIRE(blocks <= kMaxBlocks256, "too many rows for one launch");
      TGX_PROFILE("window_delta", hs);
      window_delta_kernel<T, DD><<<dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, hs>>>(
          b.a.out, static_cast<const T*>(out), static_cast<const T*>(rest), delta, rows);
      TGX_LAUNCHED("window_delta");
    }
    {
      TGX_PROFILE("window_dkdv", hs);
      b.a.tasks = k_tasks_dev;
      window_dkdv_kernel<T, DD><<<dim3(static_cast<uint32_t>(n_k_tasks)), dim3(256), 0, hs>>>(b);
      TGX_LAUNCHED("window_dkdv");
    }
    if (n_joins > 0) {
      TGX_PROFILE("window_merge", hs);
      window_merge_kernel<T, DD><<<dim3(static_cast<uint32_t>(n_joins * kMergeBlocks<DD>)),
                                   dim3(256), 0, hs>>>(b, joins_dev);
      TGX_LAUNCHED("window_merge");
    }
    {
      TGX_PROFILE("window_dq", hs);
      b.a.tasks = q_tasks_dev;
      window_dq_kernel<T, DD><<<dim3(static_cast<uint32_t>(n_q_tasks)), dim3(256), 0, hs>>>(b);
      TGX_LAUNCHED("window_dq");
    }
    return TGX_OK;
  });
}
