// Values held in 8 bits: codes of TGX_CODE_E4M3 (sign, four bits of exponent,
// three of fraction; largest 448; no infinity) or TGX_CODE_INT8 (-127 .. 127),
// which fp32, bf16 and fp16 hold exactly.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tgx.h"
#include "tgx_device.h"
#include "tgx_vals.h"

namespace tgx {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Code i of a word as fp32.
template <int CODE, int I>
__device__ __forceinline__ float code_value(uint32_t w) {
  if constexpr (CODE == TGX_CODE_E4M3) return __builtin_amdgcn_cvt_f32_fp8(w, I);
  else return static_cast<float>(static_cast<int8_t>(w >> (8 * I)));
}

template <int CODE>
__device__ __forceinline__ void widen4(uint32_t w, float* f) {
  f[0] = code_value<CODE, 0>(w);
  f[1] = code_value<CODE, 1>(w);
  f[2] = code_value<CODE, 2>(w);
  f[3] = code_value<CODE, 3>(w);
}
template <int CODE>
__device__ __forceinline__ void widen8(u32x2 w, float (&f)[8]) {
  widen4<CODE>(w[0], f);
  widen4<CODE>(w[1], f + 4);
}

// Two codes of a word (HI: the upper two) as 16-bit values.
template <typename T, int CODE, bool HI>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  if constexpr (CODE == TGX_CODE_E4M3) {
    if constexpr (__is_same(T, __bf16))
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
  } else {
    const float lo = code_value<CODE, HI ? 2 : 0>(w), hi = code_value<CODE, HI ? 3 : 1>(w);
    if constexpr (__is_same(T, __bf16))   // the upper halves: the lower ones are zero
      return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    else
      return pack_f16x2(lo, hi);
  }
}
template <typename T, int CODE>
__device__ __forceinline__ u32x4 code_octet(u32x2 w) {
  return u32x4{code_pair<T, CODE, false>(w[0]), code_pair<T, CODE, true>(w[0]),
               code_pair<T, CODE, false>(w[1]), code_pair<T, CODE, true>(w[1])};
}

// The largest code, and the power of two above it.
template <int CODE>
constexpr float kLargestCode = CODE == TGX_CODE_E4M3 ? 448.f : 127.f;
template <int CODE>
constexpr int kCodeShift = CODE == TGX_CODE_E4M3 ? 9 : 7;

// The scale of a block of largest magnitude `amax` (its bits): the smallest power
// of two s >= 2^-126 with amax <= M s; NaN for a NaN or an infinity.
template <int CODE>
__device__ __forceinline__ float block_scale(uint32_t amax) {
  if (amax >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  const float a = __uint_as_float(amax);
  // a = f 2^n, f in [1/2, 1) (n = 0 for 0).
  const float f = __builtin_amdgcn_frexp_mantf(a);
  const int n = __builtin_amdgcn_frexp_expf(a);
  const int e = n - kCodeShift<CODE> + (f > kLargestCode<CODE> / (1 << kCodeShift<CODE>));
  return __uint_as_float(static_cast<uint32_t>((a == 0.f ? -126 : max(e, -126)) + 127) << 23);
}

// Eight values times `by`, products of at most M, as codes, to the nearest, ties to
// even.  (The fused add of 1.5 * 2^23 leaves a product's nearest integer in the low
// bits, rounded once.)
template <int CODE>
__device__ __forceinline__ u32x2 encode8(const float (&f)[8], float by) {
  u32x2 w;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if constexpr (CODE == TGX_CODE_E4M3) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k] * by, f[4 * k + 1] * by, 0, false);
      v = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k + 2] * by, f[4 * k + 3] * by, v, true);
      w[k] = static_cast<uint32_t>(v);
    } else {
      uint32_t n[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        n[i] = __float_as_uint(__builtin_fmaf(f[4 * k + i], by, 12582912.f));
      w[k] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(n[3], n[2], 0x0C0C0400u),
                                   __builtin_amdgcn_perm(n[1], n[0], 0x0C0C0400u), 0x05040100u);
    }
  }
  return w;
}

// The largest magnitude among values seen, as the bits of an fp32 number (a NaN's and
// an infinity's are above all others).
template <int DT>
struct Magnitude {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 top = {0, 0};
  __device__ __forceinline__ void see(u32x4 raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, raw[i] & 0x7FFF7FFFu));
  }
  __device__ __forceinline__ uint32_t bits() const {
    const uint32_t m = max(static_cast<uint32_t>(top[0]), static_cast<uint32_t>(top[1]));
    if (DT == TGX_DTYPE_BF16) return m << 16;
    return __float_as_uint(
        static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(m))));
  }
};
template <>
struct Magnitude<TGX_DTYPE_F32> {
  uint32_t top = 0;
  __device__ __forceinline__ void see(const Vals<TGX_DTYPE_F32, 8>::Raw& raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top = max(top, __float_as_uint(raw.lo[i]) & 0x7FFFFFFFu);
      top = max(top, __float_as_uint(raw.hi[i]) & 0x7FFFFFFFu);
    }
  }
  __device__ __forceinline__ uint32_t bits() const { return top; }
};

// How a cache's rows are held: as the queries' type (code 0), or as codes.
template <int DT, int CODE>
struct CacheVals {
  using T = uint8_t;
  using Raw = u32x2;
  static __device__ __forceinline__ Raw load(const T* p) {
    return *reinterpret_cast<const u32x2*>(p);
  }
  static __device__ __forceinline__ void unpack(Raw r, float (&f)[8]) { widen8<CODE>(r, f); }
};
template <int DT>
struct CacheVals<DT, 0> : Vals<DT, 8> {};

inline bool known_code(int code) { return code == TGX_CODE_E4M3 || code == TGX_CODE_INT8; }

}  // namespace tgx
