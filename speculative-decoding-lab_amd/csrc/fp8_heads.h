// What the kernels over an 8-bit cache with head scales share.
//
// Pools hold OCP e4m3 codes in the layouts of every pool; scales are fp32
// [num_layers][num_kv_heads][capacity][2] (K, V): a code q of (layer, block,
// head) means q * scale. Heads before blocks: the allocation, which clears the
// scales of the blocks it hands out, sees num_layers * num_kv_heads layers of
// the one-scale format.
#pragma once

#include "rotary_common.h"

namespace spv {

// First byte of the (block, head) page, K or V.
__device__ __forceinline__ size_t page_of(int layer, int cap, int phys, int hkv, int h, int bs, int d) {
  return ((((size_t)layer * cap + phys) * hkv + h) * bs) * (size_t)d;
}
__device__ __forceinline__ size_t scale_of(int layer, int cap, int phys, int hkv, int h) {
  return (((size_t)layer * hkv + h) * cap + phys) * 2;
}

// Four codes of a word as fp32.
__device__ __forceinline__ void decode4(uint32_t w, float* x) {
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  x[0] = a[0];
  x[1] = a[1];
  x[2] = b[0];
  x[3] = b[1];
}

// Four values within +-448 (or NaN) as codes, to nearest even.
__device__ __forceinline__ uint32_t encode4(const float* y) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}
__device__ __forceinline__ uint8_t encode1(float y) {
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, 0.f, 0, false);
}

// x / scale as e4m3 takes it: within +-448; NaN for what is not finite (e4m3 has no infinity).
__device__ __forceinline__ float quotient(float x, float scale) {
  const float y = scale > 0.f ? fminf(fmaxf(__fdiv_rn(x, scale), -448.f), 448.f) : 0.f;
  return fabsf(x) <= 3.402823466e38f ? y : __uint_as_float(0x7fc00000u);
}

// The same for many x by one scale between 2^-60 and 2^60, by Markstein's steps: with y the rounded 1 / scale,
// q = x y is improved twice by q += (x - q scale) y, whose residual is exact; the first makes q faithful, the second
// makes it the rounded quotient. The residual of a quotient that has a code but 0 stays normal (|x| > 2^-72), and its
// form keeps the sign of a zero. 5 operations for the division's dozen.
__device__ __forceinline__ bool usual_scale(float s) { return s >= 0x1p-60f && s <= 0x1p60f; }
__device__ __forceinline__ float quotient(float x, float scale, float y) {
  float q = __fmul_rn(x, y);
  q = __fmaf_rn(-__fmaf_rn(q, scale, -x), y, q);
  q = __fmaf_rn(-__fmaf_rn(q, scale, -x), y, q);
  q = fminf(fmaxf(q, -448.f), 448.f);
  return fabsf(x) <= 3.402823466e38f ? q : __uint_as_float(0x7fc00000u);
}

// A stored code under a grown scale (grown > old >= 0): (q * old) / grown, NaN kept.
__device__ __forceinline__ float requotient(float q, float old, float grown) {
  return quotient(__fmul_rn(q, old), grown);
}

}  // namespace spv
