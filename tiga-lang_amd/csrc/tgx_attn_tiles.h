// What the dense attention tiles share (tgx_varlen.hip, tgx_window.hip): vector
// types, MFMA and lane primitives, registers of the forward.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tgx_device.h"

namespace tgx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
  typedef bf16x8 v8;
  typedef bf16x4 v4;
};
template <>
struct Vec<_Float16> {
  typedef f16x8 v8;
  typedef f16x4 v4;
};
template <typename T>
using vec8 = typename Vec<T>::v8;
template <typename T>
using vec4 = typename Vec<T>::v4;

// Workgroups per CU that a forward's registers are held to, by head dim.
template <int D>
constexpr int kFwdWaves = D == 128 ? 2 : D == 64 ? 3 : 4;
constexpr float kLog2e = 1.4426950408889634f;
// gfx950 (MI355X) has 8 XCDs, each with its own L2; workgroup i of a launch
// runs on XCD i % 8.
constexpr int kXcds = 8;

__device__ __forceinline__ f32x4v mfma(bf16x8 a, bf16x8 b, f32x4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4v mfma(f16x8 a, f16x8 b, f32x4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ vec8<T> ld8(const T* p) {
  return *reinterpret_cast<const vec8<T>*>(p);
}

// Max of a value over the four 16-lane groups (lanes l, l^16, l^32, l^48)
// with gfx950's row-swap permutes: with both operands equal, each swap
// hands every lane its partner's value in one of the two results.
__device__ __forceinline__ float group4_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                  false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x),
                                                  false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// 2^x on the hardware unit (v_exp_f32): exact 0 for -inf; results below the
// fp32 normal range flush to zero, which softmax weights tolerate.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The running max is only moved when a tile's max exceeds it by more than
// this many (log2 units): weights then stay below 2^8, exact in the final
// normalisation, and the O rescale is skipped for nearly every tile.
constexpr float kRescaleLog2 = 8.f;

}  // namespace
}  // namespace tgx
