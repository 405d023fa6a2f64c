// The 8-bit cache row, shared by the kernels that write it, read it back and attend over it.
//
// A token's row of one plane: Hkv * D e4m3 values, then Hkv * D / 32 scale bytes, one per group of
// 32 values along D, then padding.  Value i of a group with scale byte b stands for
// e4m3_i * 2^(b - 127); byte 255 stands for NaN (its values are 0).  b is the smallest exponent for
// which the group's largest magnitude fits: max|x| <= 448 * 2^(b - 127), clamped at 0; a group of
// zeros has b = 0; a group with a non-finite value has b = 255.  A power of two as scale keeps the
// products x * 2^(127 - b) and e4m3 * 2^(b - 127) exact, so the only rounding is the one to e4m3
// (nearest, ties to even; half a unit in the fourth significant bit).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace actkv {

constexpr int kQuantGroup = 32;

// 2^(b - 127) as a float; exact for b = 0 (a subnormal), NaN for b = 255.
__device__ __forceinline__ float scale_of(uint32_t b) {
  return __uint_as_float(b == 255u ? 0x7fffffffu : (b == 0u ? 0x00400000u : b << 23));
}

// Scale byte of a group whose largest magnitude has the bits `top` (sign cleared; inf / NaN -> 255).
// top = 1.m * 2^(E - 127) and 448 = 1.75 * 2^8, so the exponent is E - 8 (+ 1 when 1.m > 1.75).
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int e = int(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > 0 ? uint32_t(e) : 0u;
}

// 2^(127 - b) for the byte of a finite group (b <= 247).
__device__ __forceinline__ float inverse_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// Two e4m3 values (low byte first) as floats.
__device__ __forceinline__ float2 e4m3x2_f32(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two), __NV_E4M3);
  return __half22float2(__half2(h));
}

__device__ __forceinline__ uint32_t f32_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// A value of the cache in the type it is read in.
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) {   // past the range: its largest
  return __float2half_rn(x == x ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x);
}
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Session of packed token t, R when it is none's (before the first offset or past the last): the number of
// sessions whose last token comes at or before t.  Called by a whole warp with one t; 32 offsets per step.
__device__ __forceinline__ int session_of(const int32_t* off, int R, int t, int lane) {
  int n = 0;
  for (int base = 0; base < R; base += 32) {
    const bool before = base + lane < R && off[base + lane + 1] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, before));
    n += c;
    if (c < 32) break;
  }
  return n < R && t >= off[n] ? n : R;
}

}  // namespace actkv
