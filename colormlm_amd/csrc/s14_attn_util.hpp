// Device helpers of the attention kernels (s14_attn_*.hip).  Unnamed
// namespace: each kernel file gets its own inline copy.
#pragma once

#include <hip/hip_runtime.h>

#include "s14_attn.hpp"

namespace s14 {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRise = 8.0f;  // how far (log2) a maximum may pass the one that weights are taken from

// A row bound from device memory, held inside the packed rows.
__device__ __forceinline__ int64_t clamp_row(int32_t r, uint32_t rows) {
  return r < 0 ? 0 : int64_t(r) > int64_t(rows) ? int64_t(rows) : int64_t(r);
}

__device__ __forceinline__ float power_of_two(int e) { return __builtin_ldexpf(1.0f, e); }

// a and b rounded to bf16 (ties to even, NaN stays NaN), a in the low half.
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}

// The positions a row sees, base .. base + count - 1: those up to its own, of
// a window the last ones.  One unsigned comparison answers for a position.
// (Masks are selects of plain floats everywhere: writing an element of a
// matrix result in a divergent branch has been compiled into a copy of that
// element over its neighbours, clang 20 of ROCm 7.2, when registers spill.)
struct Visible {
  int32_t base;
  uint32_t count;
  __device__ __forceinline__ Visible(int32_t pos, uint32_t window) {
    base = window && pos >= 0 && window <= uint32_t(pos) ? pos - int32_t(window) + 1 : 0;
    count = pos < 0 ? 0u : uint32_t(pos - base) + 1u;
  }
  Visible() = default;
  __device__ __forceinline__ bool operator()(int32_t j) const { return uint32_t(j - base) < count; }
};

// Inside a uniform branch: it stays one.  (A mask's selects are otherwise done
// in every step, taken or not: a third of the softmax's instructions.)
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// A row's sum of weights taken from the maximum top (log2), NaN where top is 2^29
// or more in magnitude (-inf, nothing seen, is not): the weights' exponents are
// x * scale - top with one rounding, so that the largest is off by top's own
// rounding, 2^5 there; further up it would be 0 or infinite, and the row 0 as if
// it saw nothing.  (Asked once a row: where the maximum moves it took 3 % of 32
// sequences of 8 new and 300 tokens.)
__device__ __forceinline__ float checked_sum(float sum, float top) {
  return fabsf(top) >= 0x1p29f && top != -INFINITY ? __uint_as_float(0x7fc00000u) : sum;
}

// The result of a max or sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_lane16(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_lane16(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Eight E4M3 codes times a power of two as bf16, exactly within bf16's range (a
// NaN code gives NaN).
__device__ __forceinline__ bf16x8 e4m3_bf16(uint32_t lo, uint32_t hi, float scale = 1.0f) {
  const u32x4 v = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
  return __builtin_bit_cast(bf16x8, v);
}

}  // namespace
}  // namespace s14
