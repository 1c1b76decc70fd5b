// 8-bit cache rows with one scale per (token, KV head), shared by the append
// and the decode kernels.
//
// A row x of head_dim values is held as codes c_d and a scale s, x_d ~ s c_d:
//     a = max_d |x_d|,  s = a / top,  c_d = round(x_d * (top * (1 / a))),
// top = 127 (int8, round to nearest even, clamped to +-127) or 448 (e4m3, the
// conversion's round to nearest even, saturating).  The factor top * (1 / a)
// and the product with it round to fp32: at most 3 * 2^-24 of the value before
// it is rounded to 8 bits, for one division per row instead of head_dim.  Rows whose largest magnitude is
// below 2^-100 are stored as zeros with scale 0 (their reciprocal overflows);
// a row with an infinity or NaN gets scale NaN, so whatever attends to it
// reads NaN.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace clover {

// |x| as an integer that orders like the magnitude, with NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of a row and the factor its values take, from max |x| (as bits).
__device__ __forceinline__ float row_scale(uint32_t amax_bits, float top, float& factor) {
  const float a = __uint_as_float(amax_bits);
  factor = 0.f;
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if (a < 7.8886090522101181e-31f) return 0.f;  // 2^-100
  factor = __fmul_rn(__frcp_rn(a), top);
  return __fdiv_rn(a, top);
}

template <bool FP8>
__device__ __forceinline__ float code_top() { return FP8 ? 448.f : 127.f; }

// Four codes in one word, lowest index in the lowest byte.  factor = 0 (a zero
// or non-finite row) gives zeros.
template <bool FP8>
__device__ __forceinline__ uint32_t encode4(const float* x, float factor) {
  if (factor == 0.f) return 0u;
  if (FP8) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * factor, x[1] * factor), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * factor, x[3] * factor), __NV_SATFINITE, __NV_E4M3);
    return (lo & 0xffffu) | (hi << 16);
  }
  // Adding 1.5 * 2^23 leaves the value rounded to nearest even in the low bits
  // (|x factor| is at most 127 (1 + 3 * 2^-24): 127 after rounding, no clamp).
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], factor), 12582912.f));
  return __byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410);
}

template <bool FP8>
__device__ __forceinline__ uint8_t encode1(float x, float factor) {
  if (factor == 0.f) return 0;
  if (FP8) return __nv_cvt_float_to_fp8(x * factor, __NV_SATFINITE, __NV_E4M3);
  const int v = max(-127, min(127, __float2int_rn(x * factor)));
  return (uint8_t)(v & 0xff);
}

// One row by one warp, any head_dim: codes to dst[0, D), returns the scale (on
// every lane).
template <bool FP8, typename TI>
__device__ __forceinline__ float encode_row_warp(const TI* src, uint8_t* dst, int D, int lane) {
  uint32_t m = 0;
  for (int d = lane; d < D; d += 32) m = max(m, abs_bits(load_f<TI>(src + d)));
  m = __reduce_max_sync(0xffffffffu, m);
  float f;
  const float s = row_scale(m, code_top<FP8>(), f);
  for (int d = lane; d < D; d += 32) dst[d] = encode1<FP8>(load_f<TI>(src + d), f);
  return s;
}

// The same for a row of any type at element `at` of src.
template <bool FP8>
__device__ __forceinline__ float encode_row_any(int dtype, const void* src, int64_t at, uint8_t* dst,
                                                int D, int lane) {
  switch (dtype) {
    case CLOVER_B200_F32: return encode_row_warp<FP8>(static_cast<const float*>(src) + at, dst, D, lane);
    case CLOVER_B200_F16: return encode_row_warp<FP8>(static_cast<const __half*>(src) + at, dst, D, lane);
    default: return encode_row_warp<FP8>(static_cast<const __nv_bfloat16*>(src) + at, dst, D, lane);
  }
}

}  // namespace clover
