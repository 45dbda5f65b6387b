// RMS norm of every head's query or key and the rotation by its token's
// positions, in one pass, with gradients (tg.nn.norm_rotary).
//
// For a row x of D values (one token, one head), with n_freqs = R / 2:
//
//   r = (mean_d x_d^2 + eps)^(-1/2),  n = r x,  u = w n      (norm; else u = x)
//   theta_i = position[axis(i)] * frequency_i                 i < R / 2
//   y_a = u_a cos theta_i - u_b sin theta_i
//   y_b = u_b cos theta_i + u_a sin theta_i                   (a, b) the i-th pair
//
// pairs are (i, i + R / 2), or (2 i, 2 i + 1) when interleaved; values from R
// on are not rotated.  With g the pairs of dy rotated back:
//
//   dw = sum over tokens and heads of g n,   h = w g,
//   dx = r (h - n mean_d(h_d n_d))
//
// All of it in fp32 but the angle, which is reduced in fp64: at position 10^6
// an fp32 angle is off by 0.03.
//
// Bound: x is read and y written once (backward: x and dy read, dx written)
// against some 20 operations a value: memory.  A lane holds one chunk of each
// half of the pairs (2 N values), LPR lanes a row, a wave 64 / LPR rows; the
// sines of a token are formed once for all of its rows in the wave.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "tgx_device.h"
#include "tgx_host.h"
#include "tgx_profile.h"
#include "tgx_vals.h"

namespace tgx {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

struct RotaryArgs {
  const void* x[2];         // queries, keys
  int64_t xs_token[2], xs_head[2];
  const void* dy[2];        // backward: contiguous [tokens, heads, D]
  void* out[2];             // y, or dx: contiguous
  const void* w[2];         // [D], null: ones
  int heads[2];
  const void* positions;    // [tokens, axes]
  int wide_positions;       // int64, else int32
  int axes;
  int ends[4];              // frequencies before the end of each axis
  const float* freqs;
  int half;                 // R / 2
  int64_t tokens;
  int split;                // waves that share a token's rows
  int D;
  float eps;
  int norm;
  int w_dtype;
  float* partial;           // backward: [workgroup, 2, D] sums of g n; null: not wanted
};

template <int DT, int N>
struct Chunk;
template <int DT>
struct Chunk<DT, 8> {
  using V = Vals<DT, 8>;
  using T = typename V::T;
  using Raw = typename V::Raw;
  static __device__ __forceinline__ Raw load(const T* p) { return V::load(p); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[8]) { V::unpack(r, f); }
  // FAR: past the caches, for outputs that they would not hold anyway.
  template <bool FAR>
  static __device__ __forceinline__ void store(T* p, const float (&f)[8]) {
    if constexpr (!FAR) {
      V::store(p, f);
    } else if constexpr (DT == TGX_DTYPE_F32) {
      f32x4* q = reinterpret_cast<f32x4*>(p);
      __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, q);
      __builtin_nontemporal_store(f32x4{f[4], f[5], f[6], f[7]}, q + 1);
    } else {
      u32x4 w;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = DT == TGX_DTYPE_BF16 ? pack_bf16x2(f[2 * k], f[2 * k + 1])
                                    : pack_f16x2(f[2 * k], f[2 * k + 1]);
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
    }
  }
};
template <>
struct Chunk<TGX_DTYPE_F32, 2> {
  using T = float;
  typedef float Raw __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ Raw load(const T* p) {
    return *reinterpret_cast<const Raw*>(p);
  }
  static __device__ __forceinline__ void unpack(Raw r, float (&f)[2]) {
    f[0] = r[0];
    f[1] = r[1];
  }
  template <bool>
  static __device__ __forceinline__ void store(T* p, const float (&f)[2]) {
    *reinterpret_cast<Raw*>(p) = Raw{f[0], f[1]};
  }
};
template <>
struct Chunk<TGX_DTYPE_BF16, 2> {
  using T = uint16_t;
  using Raw = uint32_t;
  static __device__ __forceinline__ Raw load(const T* p) {
    return *reinterpret_cast<const uint32_t*>(p);
  }
  static __device__ __forceinline__ void unpack(Raw r, float (&f)[2]) {
    f[0] = bf16_lo(r);
    f[1] = bf16_hi(r);
  }
  template <bool>
  static __device__ __forceinline__ void store(T* p, const float (&f)[2]) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(f[0], f[1]);
  }
};
template <>
struct Chunk<TGX_DTYPE_F16, 2> {
  using T = uint16_t;
  using Raw = uint32_t;
  static __device__ __forceinline__ Raw load(const T* p) {
    return *reinterpret_cast<const uint32_t*>(p);
  }
  static __device__ __forceinline__ void unpack(Raw r, float (&f)[2]) { f16_pair(r, f[0], f[1]); }
  template <bool>
  static __device__ __forceinline__ void store(T* p, const float (&f)[2]) {
    *reinterpret_cast<uint32_t*>(p) = pack_f16x2(f[0], f[1]);
  }
};

__device__ __forceinline__ float scalar_value(const void* p, int dtype, int i) {
  if (dtype == TGX_DTYPE_F32) return static_cast<const float*>(p)[i];
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  return dtype == TGX_DTYPE_BF16 ? bf16_lo(u) : static_cast<float>(__builtin_bit_cast(_Float16, u));
}
__device__ __forceinline__ void store_scalar(void* p, int dtype, int i, float v) {
  if (dtype == TGX_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == TGX_DTYPE_BF16)
    static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(f32_to_bf16_bits(v));
  else static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}

// Where a lane's two chunks of a row are, so that the lanes of a row take one
// run of columns with each: the two halves of the rotated columns and of the
// rest, or (adjacent pairs) of the row.  The lane's pair j is frequency `low` +
// j, from j = N / 2 on `high` + j; pairs of columns that are not rotated
// have frequencies from n_freqs on.
template <int N, bool INTER>
struct Place {
  int first, second;   // columns of the chunks
  int low, high;
  bool has;
  __device__ __forceinline__ Place(const RotaryArgs& a, int part) {
    has = 2 * N * part < a.D;
    if constexpr (INTER) {
      first = N * part;
      second = a.D / 2 + N * part;
      low = N / 2 * part;
      high = a.D / 4 + N / 2 * part - N / 2;
    } else {
      const int c = N * part;
      first = c < a.half ? c : c + a.half;
      second = c < a.half ? c + a.half : c + a.D / 2;
      low = high = c;
    }
    if (!has) low = high = 0;
  }
};

// cos and sin of the token's angles, [pair][2] in `cs` (LDS of the wave): a
// lane forms every 64th pair's, and all lanes read those of their own pairs.
// Pairs past the rotated ones turn by nothing.
template <int PAIRS>
__device__ __forceinline__ void form_turns(const RotaryArgs& a, int64_t token,
                                           const float (&freq)[PAIRS / 64 + 1], float* cs) {
#pragma unroll
  for (int k = 0; 64 * k < PAIRS; ++k) {
    const int i = 64 * k + lane_id();
    if (PAIRS % 64 && i >= PAIRS) break;
    float sn = 0.f, c = 1.f;
    if (i < a.half) {
      const int axis = (i >= a.ends[0]) + (i >= a.ends[1]) + (i >= a.ends[2]);
      const int64_t at = token * a.axes + axis;
      const double pos = a.wide_positions
                             ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                             : static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
      // The angle in half turns, without the whole turns; what its fp32 value
      // leaves is put back to first order.
      const double t = pos * static_cast<double>(freq[k]) * 0.15915494309189535;
      const double u = 2.0 * (t - __builtin_rint(t));
      const float uf = static_cast<float>(u);
      const float rest = static_cast<float>((u - static_cast<double>(uf)) * 3.141592653589793);
      float s0, c0;
      sincospif(uf, &s0, &c0);
      c = fmaf(-s0, rest, c0);
      sn = fmaf(c0, rest, s0);
    }
    cs[2 * i] = c;
    cs[2 * i + 1] = sn;
  }
}

// The turns of the lane's pairs.
template <int N, bool INTER>
__device__ __forceinline__ void read_turns(const float* cs, const Place<N, INTER>& at,
                                           float (&c)[N], float (&s)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const f32x2 v = *reinterpret_cast<const f32x2*>(cs + 2 * ((j < N / 2 ? at.low : at.high) + j));
    c[j] = v[0];
    s[j] = v[1];
  }
}

// 1 / sqrt(v): the hardware's value and one Newton step.  The hardware takes
// subnormal numbers for 0 (eps = 0 and rows of values below 2^-63), so those
// are multiplied by an even power of two first.
__device__ __forceinline__ float inverse_root(float v) {
  const bool small = v < 0x1p-126f;
  const float u = small ? v * 0x1p64f : v;
  const float r = __builtin_amdgcn_rsqf(u);
  // (u = 0 or Inf: r is Inf or 0, and stays.)
  const float e = fmaf(-u * r, r, 1.f);
  const float root = u > 0.f && u < __builtin_huge_valf() ? fmaf(0.5f * r, e, r) : r;
  return small ? root * 0x1p32f : root;
}

// Turns pair j of the chunks (f, g) by (c, s): the halves of the pairs lie in
// f and g, or next to each other.  Pairs that are not rotated stay as they are
// (turning them by nothing would multiply one's Inf by the other's sine of 0).
template <int N, bool INTER>
__device__ __forceinline__ void rotate(const RotaryArgs& a, const Place<N, INTER>& at,
                                       float (&f)[N], float (&g)[N], const float (&c)[N],
                                       const float (&s)[N], float sign) {
  // (Apart, a lane's pairs are all rotated or none: half is a multiple of N.)
  if (!INTER && at.low >= a.half) return;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float* pa = INTER ? (j < N / 2 ? &f[2 * j] : &g[2 * j - N]) : &f[j];
    float* pb = INTER ? pa + 1 : &g[j];
    const float x = *pa, y = *pb, sj = sign * s[j];
    const bool turns = !INTER || (j < N / 2 ? at.low : at.high) + j < a.half;
    *pa = turns ? x * c[j] - y * sj : x;
    *pb = turns ? y * c[j] + x * sj : y;
  }
}

template <int N>
struct Weights {
  float f[2][N], g[2][N];
  template <bool INTER>
  __device__ __forceinline__ void load(const RotaryArgs& a, const Place<N, INTER>& at) {
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const bool have = a.norm && a.w[side] && at.has;
        f[side][j] = have ? scalar_value(a.w[side], a.w_dtype, at.first + j) : 1.f;
        g[side][j] = have ? scalar_value(a.w[side], a.w_dtype, at.second + j) : 1.f;
      }
  }
};

// Passes of 64 / LPR rows whose loads are issued together.
constexpr int kPasses = 2;

template <int DT, int N, int LPR, bool INTER, bool FAR>
__global__ __launch_bounds__(256) void norm_rotary_fwd_kernel(RotaryArgs a) {
  using C = Chunk<DT, N>;
  using T = typename C::T;
  constexpr int RPP = 64 / LPR, PAIRS = N * LPR;
  __shared__ __align__(16) float turns[4][2 * PAIRS];
  float* cs = turns[threadIdx.x >> 6];
  const int lane = lane_id(), part = lane % LPR, sub = lane / LPR;
  const Place<N, INTER> at(a, part);
  Weights<N> w;
  w.load(a, at);
  float freq[PAIRS / 64 + 1];
#pragma unroll
  for (int k = 0; 64 * k < PAIRS; ++k) freq[k] = 64 * k + lane < a.half ? a.freqs[64 * k + lane] : 0.f;
  const int rows = a.heads[0] + a.heads[1];
  const int64_t items = a.tokens * a.split;
  const float inv_d = 1.f / static_cast<float>(a.D);
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); item < items;
       item += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t token = item / a.split;
    const int step = a.split * RPP;
    float c[N], s[N];
    bool formed = false;
    for (int row0 = static_cast<int>(item % a.split) * RPP + sub; row0 - sub < rows;
         row0 += kPasses * step) {
      typename C::Raw first[kPasses], second[kPasses];
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int row = row0 + p * step;
        const int side = row >= a.heads[0];
        if (row < rows && at.has) {
          const T* x = static_cast<const T*>(a.x[side]) + token * a.xs_token[side] +
                       (row - (side ? a.heads[0] : 0)) * a.xs_head[side];
          first[p] = C::load(x + at.first);
          second[p] = C::load(x + at.second);
        } else {
          first[p] = typename C::Raw{};
          second[p] = typename C::Raw{};
        }
      }
      if (!formed) {
        form_turns<PAIRS>(a, token, freq, cs);
        __builtin_amdgcn_wave_barrier();
        read_turns<N, INTER>(cs, at, c, s);
        formed = true;
      }
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int row = row0 + p * step;
        if (row - sub >= rows) break;
        const int side = row >= a.heads[0];
        float f[N], g[N];
        C::unpack(first[p], f);
        C::unpack(second[p], g);
        if (a.norm) {
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < N; ++j) ss += f[j] * f[j] + g[j] * g[j];
          const float r = inverse_root(group_sum<LPR>(ss) * inv_d + a.eps);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            f[j] *= r * (side ? w.f[1][j] : w.f[0][j]);
            g[j] *= r * (side ? w.g[1][j] : w.g[0][j]);
          }
        }
        rotate<N, INTER>(a, at, f, g, c, s, 1.f);
        if (row < rows && at.has) {
          T* y = static_cast<T*>(a.out[side]) +
                 (token * a.heads[side] + row - (side ? a.heads[0] : 0)) * a.D;
          C::template store<FAR>(y + at.first, f);
          C::template store<FAR>(y + at.second, g);
        }
      }
    }
  }
}

constexpr int kBwdPasses = 1;

template <int DT, int N, int LPR, bool INTER, bool FAR>
__global__ __launch_bounds__(256) void norm_rotary_bwd_kernel(RotaryArgs a) {
  using C = Chunk<DT, N>;
  using T = typename C::T;
  constexpr int RPP = 64 / LPR, PAIRS = N * LPR;
  __shared__ __align__(16) float turns[4][2 * PAIRS];
  float* cs = turns[threadIdx.x >> 6];
  const int lane = lane_id(), part = lane % LPR, sub = lane / LPR;
  const Place<N, INTER> at(a, part);
  Weights<N> w;
  w.load(a, at);
  float freq[PAIRS / 64 + 1];
#pragma unroll
  for (int k = 0; 64 * k < PAIRS; ++k) freq[k] = 64 * k + lane < a.half ? a.freqs[64 * k + lane] : 0.f;
  float wf[2][N], wg[2][N];   // sums of g n
#pragma unroll
  for (int j = 0; j < N; ++j) wf[0][j] = wf[1][j] = wg[0][j] = wg[1][j] = 0.f;
  const int64_t items = a.tokens * a.split;
  const float inv_d = 1.f / static_cast<float>(a.D);
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); item < items;
       item += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t token = item / a.split;
    const int step = a.split * RPP;
    float c[N], s[N];
    bool formed = false;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int heads = a.heads[side];
      for (int head0 = static_cast<int>(item % a.split) * RPP + sub; head0 - sub < heads;
           head0 += kBwdPasses * step) {
        typename C::Raw x1[kBwdPasses], x2[kBwdPasses], d1[kBwdPasses], d2[kBwdPasses];
#pragma unroll
        for (int p = 0; p < kBwdPasses; ++p) {
          const int head = head0 + p * step;
          if (head < heads && at.has) {
            const T* x = static_cast<const T*>(a.x[side]) + token * a.xs_token[side] +
                         head * a.xs_head[side];
            const T* dy = static_cast<const T*>(a.dy[side]) + (token * heads + head) * a.D;
            x1[p] = C::load(x + at.first);
            x2[p] = C::load(x + at.second);
            d1[p] = C::load(dy + at.first);
            d2[p] = C::load(dy + at.second);
          } else {
            x1[p] = x2[p] = d1[p] = d2[p] = typename C::Raw{};
          }
        }
        if (!formed) {
          form_turns<PAIRS>(a, token, freq, cs);
          __builtin_amdgcn_wave_barrier();
          read_turns<N, INTER>(cs, at, c, s);
          formed = true;
        }
#pragma unroll
        for (int p = 0; p < kBwdPasses; ++p) {
          const int head = head0 + p * step;
          if (head - sub >= heads) break;
          float f[N], g[N], df[N], dg[N];
          C::unpack(x1[p], f);
          C::unpack(x2[p], g);
          C::unpack(d1[p], df);
          C::unpack(d2[p], dg);
          rotate<N, INTER>(a, at, df, dg, c, s, -1.f);
          if (a.norm) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) ss += f[j] * f[j] + g[j] * g[j];
            const float r = inverse_root(group_sum<LPR>(ss) * inv_d + a.eps);
            float hn = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
              f[j] *= r;
              g[j] *= r;
              // (A row that is not there is zero, and with eps = 0 its r is Inf.)
              if (head < heads) {
                wf[side][j] += df[j] * f[j];
                wg[side][j] += dg[j] * g[j];
              }
              df[j] *= w.f[side][j];
              dg[j] *= w.g[side][j];
              hn += df[j] * f[j] + dg[j] * g[j];
            }
            hn = group_sum<LPR>(hn) * inv_d;
#pragma unroll
            for (int j = 0; j < N; ++j) {
              df[j] = r * (df[j] - f[j] * hn);
              dg[j] = r * (dg[j] - g[j] * hn);
            }
          }
          if (head < heads && at.has) {
            T* dx = static_cast<T*>(a.out[side]) + (token * heads + head) * a.D;
            C::template store<FAR>(dx + at.first, df);
            C::template store<FAR>(dx + at.second, dg);
          }
        }
      }
    }
  }
  if (!a.partial) return;
  // The rows of a wave, then the four waves, in a fixed order.
  __shared__ float sums[4][2][2 * N * LPR];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int j = 0; j < N; ++j) {
#pragma unroll
      for (int mask = LPR; mask < 64; mask <<= 1) {
        wf[side][j] += __shfl_xor(wf[side][j], mask, 64);
        wg[side][j] += __shfl_xor(wg[side][j], mask, 64);
      }
      if (sub == 0 && at.has) {
        sums[threadIdx.x >> 6][side][at.first + j] = wf[side][j];
        sums[threadIdx.x >> 6][side][at.second + j] = wg[side][j];
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.D; i += 256) {
    const int side = i / a.D, d = i % a.D;
    a.partial[static_cast<int64_t>(blockIdx.x) * 2 * a.D + i] =
        (sums[0][side][d] + sums[1][side][d]) + (sums[2][side][d] + sums[3][side][d]);
  }
}

// dw[side][d] = sum over the workgroups of the backward: 16 columns a
// workgroup, 64 threads on each, whole 64-byte lines a load.
__global__ __launch_bounds__(1024) void norm_rotary_dw_kernel(const float* partial, int blocks,
                                                              int D, int dtype, void* dwq,
                                                              void* dwk) {
  __shared__ float sums[64][17];
  const int col = threadIdx.x % 16, part = threadIdx.x / 16;
  const int i = blockIdx.x * 16 + col;
  float s = 0.f;
  if (i < 2 * D) {
#pragma unroll 8
    for (int b = part; b < blocks; b += 64) s += partial[static_cast<int64_t>(b) * 2 * D + i];
  }
  sums[part][col] = s;
  __syncthreads();
  if (threadIdx.x >= 64 * 16 / 4) return;
  // Wave w adds the columns 4 w .. 4 w + 3.
  const int wave = threadIdx.x >> 6, lane = lane_id();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = 4 * wave + k, at = blockIdx.x * 16 + c;
    const float total = group_sum<64>(sums[lane][c]);
    void* out = at < D ? dwq : dwk;
    if (lane == 0 && at < 2 * D && out) store_scalar(out, dtype, at % D, total);
  }
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Outputs of more bytes than this are stored past the caches (a fraction of
// the last level, so that what reads a smaller one next finds it there): 16384
// tokens of 32 + 8 heads of 128, bf16, forward and backward 187 -> 160 us.
constexpr int64_t kCached = int64_t{64} << 20;

// Workgroups at most: enough to fill the GPU, few enough that the weights and
// frequencies a wave loads first serve many tokens.
constexpr int64_t kFwdBlocks = 1024;
constexpr int64_t kBwdBlocks = 512;

// Waves that share a token's rows: with few tokens, so many that the rows of a
// token do not queue behind each other.
int rows_split(const tgx_norm_rotary& p, int rows_per_wave) {
  const int passes = (std::max(p.heads[0], 1) + p.heads[1] + rows_per_wave - 1) / rows_per_wave;
  if (p.n_tokens >= 4096) return 1;
  return static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(passes, 4096 / std::max<int64_t>(p.n_tokens, 1))));
}

struct Form {
  int n;     // values a chunk
  int lpr;   // lanes a row
};

Form form_of(const tgx_norm_rotary& p, bool wide) {
  // Chunks of 8 values where the pairs divide into them and every row starts
  // on 16 bytes, of 2 elsewhere.
  const bool eight = wide && p.D % 16 == 0 && (p.interleaved || p.n_freqs % 8 == 0);
  if (!eight) return Form{2, 64};
  const int lanes = p.D / 16;
  return Form{8, lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16};
}

int check(const tgx_norm_rotary* p) {
  TGX_REQUIRE(p != nullptr, "null operands");
  TGX_REQUIRE(dtype_bytes(p->dtype) != 0 && dtype_bytes(p->w_dtype) != 0, "unknown dtype");
  TGX_REQUIRE(p->n_tokens >= 0 && p->heads[0] >= 0 && p->heads[1] >= 0, "negative sizes");
  if (p->D < 4 || p->D > 256 || p->D % 4 || p->n_freqs % 2) {
    set_error("head width %d with %d frequencies: norm_rotary takes widths that are multiples of "
              "4 up to 256 and an even number of frequencies", p->D, p->n_freqs);
    return TGX_UNSUPPORTED;
  }
  TGX_REQUIRE(p->n_freqs >= 0 && 2 * p->n_freqs <= p->D, "more frequencies than pairs");
  TGX_REQUIRE(p->axes >= 1 && p->axes <= 4, "1 to 4 position axes");
  int total = 0;
  for (int i = 0; i < p->axes; ++i) {
    TGX_REQUIRE(p->sections[i] >= 0, "negative section");
    total += p->sections[i];
  }
  TGX_REQUIRE(total == p->n_freqs, "sections cover %d of %d frequencies", total, p->n_freqs);
  TGX_REQUIRE(p->n_tokens == 0 || p->n_freqs == 0 || (p->positions_dev && p->freqs_dev),
              "null positions or frequencies");
  TGX_REQUIRE(p->positions_bits == 32 || p->positions_bits == 64, "positions are 32 or 64 bits");
  for (int i = 0; i < 2; ++i)
    TGX_REQUIRE(p->n_tokens == 0 || p->heads[i] == 0 || p->x_dev[i], "null input");
  return TGX_OK;
}

// Fills the kernels' arguments; `wide`: all rows on 16 bytes (else on two values).
int args_of(const tgx_norm_rotary& p, void* const out[2], const void* const dy[2], RotaryArgs* a,
            bool* wide) {
  const int size = dtype_bytes(p.dtype);
  *wide = true;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0 || p.n_tokens == 0) continue;
    TGX_REQUIRE(out[i] && (!dy || dy[i]), "null output or gradient");
    const void* ptrs[3] = {p.x_dev[i], out[i], dy ? dy[i] : out[i]};
    for (const void* q : ptrs) {
      TGX_REQUIRE(aligned(q, 2 * size), "rows must start on two values");
      *wide = *wide && aligned(q, 16);
    }
    TGX_REQUIRE(p.token_stride[i] % 2 == 0 && p.head_stride[i] % 2 == 0,
                "rows must start on two values");
    *wide = *wide && p.token_stride[i] * size % 16 == 0 && p.head_stride[i] * size % 16 == 0 &&
            p.D * size % 16 == 0;
    a->x[i] = p.x_dev[i];
    a->xs_token[i] = p.token_stride[i];
    a->xs_head[i] = p.head_stride[i];
    a->out[i] = out[i];
    a->dy[i] = dy ? dy[i] : nullptr;
  }
  int end = 0;
  for (int i = 0; i < 4; ++i) {
    end += i < p.axes ? p.sections[i] : 0;
    // Axes past the last never start.
    a->ends[i] = i + 1 < p.axes ? end : 1 << 30;
  }
  for (int i = 0; i < 2; ++i) {
    a->w[i] = p.w_dev[i];
    a->heads[i] = p.heads[i];
  }
  a->positions = p.positions_dev;
  a->wide_positions = p.positions_bits == 64;
  a->axes = p.axes;
  a->freqs = p.freqs_dev;
  a->half = p.n_freqs;
  a->tokens = p.n_tokens;
  a->D = p.D;
  a->eps = p.eps;
  a->norm = p.norm;
  a->w_dtype = p.w_dtype;
  return TGX_OK;
}

template <bool BWD, int DT, int N, int LPR, bool FAR>
int launch(const RotaryArgs& a, bool inter, int64_t blocks, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(blocks)), block(256);
  if constexpr (BWD) {
    TGX_PROFILE("norm_rotary_bwd", stream);
    if (inter) norm_rotary_bwd_kernel<DT, N, LPR, true, FAR><<<grid, block, 0, stream>>>(a);
    else norm_rotary_bwd_kernel<DT, N, LPR, false, FAR><<<grid, block, 0, stream>>>(a);
  } else {
    TGX_PROFILE("norm_rotary_fwd", stream);
    if (inter) norm_rotary_fwd_kernel<DT, N, LPR, true, FAR><<<grid, block, 0, stream>>>(a);
    else norm_rotary_fwd_kernel<DT, N, LPR, false, FAR><<<grid, block, 0, stream>>>(a);
  }
  TGX_LAUNCHED(BWD ? "norm_rotary_bwd" : "norm_rotary_fwd");
  return TGX_OK;
}

template <bool BWD, int DT, int LPR>
int launch_wide(const RotaryArgs& a, bool far, bool inter, int64_t blocks, hipStream_t s) {
  return far ? launch<BWD, DT, 8, LPR, true>(a, inter, blocks, s)
             : launch<BWD, DT, 8, LPR, false>(a, inter, blocks, s);
}

template <bool BWD, int DT>
int by_form(const RotaryArgs& a, Form f, bool far, bool inter, int64_t blocks, hipStream_t s) {
  if (f.n == 2) return launch<BWD, DT, 2, 64, false>(a, inter, blocks, s);
  switch (f.lpr) {
    case 2: return launch_wide<BWD, DT, 2>(a, far, inter, blocks, s);
    case 4: return launch_wide<BWD, DT, 4>(a, far, inter, blocks, s);
    case 8: return launch_wide<BWD, DT, 8>(a, far, inter, blocks, s);
    default: return launch_wide<BWD, DT, 16>(a, far, inter, blocks, s);
  }
}

template <bool BWD>
int run(const tgx_norm_rotary& p, RotaryArgs a, bool wide, int64_t max_blocks, hipStream_t s) {
  const Form f = form_of(p, wide);
  a.split = rows_split(p, 64 / f.lpr);
  const int size = dtype_bytes(p.dtype);
  // (Lines that a store instruction fills only in part belong in the caches.)
  const int runs[2] = {p.interleaved ? p.D / 2 : p.n_freqs, p.interleaved ? 0 : p.D / 2 - p.n_freqs};
  const bool far = p.n_tokens * (p.heads[0] + p.heads[1]) * p.D * size > kCached &&
                   runs[0] * size % 128 == 0 && runs[1] * size % 128 == 0;
  const int64_t blocks = std::min(max_blocks, ceil_div(p.n_tokens * a.split, 4));
  switch (p.dtype) {
    case TGX_DTYPE_BF16: return by_form<BWD, TGX_DTYPE_BF16>(a, f, far, p.interleaved, blocks, s);
    case TGX_DTYPE_F16: return by_form<BWD, TGX_DTYPE_F16>(a, f, far, p.interleaved, blocks, s);
    default: return by_form<BWD, TGX_DTYPE_F32>(a, f, far, p.interleaved, blocks, s);
  }
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_norm_rotary_fwd(const tgx_norm_rotary* p, void* query_out_dev,
                                   void* key_out_dev, void* stream) {
  if (int st = check(p)) return st;
  if (p->n_tokens == 0 || p->heads[0] + p->heads[1] == 0) return TGX_OK;
  void* const out[2] = {query_out_dev, key_out_dev};
  RotaryArgs a{};
  bool wide = true;
  if (int st = args_of(*p, out, nullptr, &a, &wide)) return st;
  return run<false>(*p, a, wide, kFwdBlocks, as_stream(stream));
}

extern "C" int tgx_norm_rotary_bwd_workspace(const tgx_norm_rotary* p, size_t* bytes) {
  TGX_REQUIRE(bytes != nullptr, "null bytes");
  if (int st = check(p)) return st;
  *bytes = sizeof(float) * kBwdBlocks * 2 * p->D;
  return TGX_OK;
}

extern "C" int tgx_norm_rotary_bwd(const tgx_norm_rotary* p, const void* dquery_out_dev,
                                   const void* dkey_out_dev, void* dquery_dev, void* dkey_dev,
                                   void* dquery_weight_dev, void* dkey_weight_dev,
                                   void* workspace_dev, size_t workspace_bytes, void* stream) {
  if (int st = check(p)) return st;
  const bool weights = p->norm && (dquery_weight_dev || dkey_weight_dev);
  const bool work = p->n_tokens > 0 && p->heads[0] + p->heads[1] > 0;
  if (!work && !weights) return TGX_OK;
  void* const out[2] = {dquery_dev, dkey_dev};
  const void* const dy[2] = {dquery_out_dev, dkey_out_dev};
  RotaryArgs a{};
  bool wide = true;
  if (int st = args_of(*p, out, dy, &a, &wide)) return st;
  const int64_t max_blocks = kBwdBlocks;
  const Form f = form_of(*p, wide);
  const int64_t blocks =
      work ? std::min(max_blocks, ceil_div(p->n_tokens * rows_split(*p, 64 / f.lpr), 4)) : 0;
  if (weights) {
    TGX_REQUIRE(workspace_dev && workspace_bytes >= sizeof(float) * blocks * 2 * p->D,
                "workspace too small");
    a.partial = static_cast<float*>(workspace_dev);
  }
  if (work)
    if (int st = run<true>(*p, a, wide, max_blocks, as_stream(stream))) return st;
  if (weights) {
    {
      TGX_PROFILE("norm_rotary_dw", as_stream(stream));
      norm_rotary_dw_kernel<<<dim3(static_cast<uint32_t>(ceil_div(2 * p->D, 16))), dim3(1024), 0,
                              as_stream(stream)>>>(a.partial, static_cast<int>(blocks), p->D,
                                                   p->w_dtype, dquery_weight_dev,
                                                   dkey_weight_dev);
    }
    TGX_LAUNCHED("norm_rotary_dw");
  }
  return TGX_OK;
}
