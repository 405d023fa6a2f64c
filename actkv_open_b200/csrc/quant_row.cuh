// The rows of the 8-bit and the 4-bit cache, shared by the kernels that write them, read them back and
// attend over them.
//
// A token's row of one plane: Hkv * D e4m3 values, then Hkv * D / 32 scale bytes, one per group of
// 32 values along D, then padding.  Value i of a group with scale byte b stands for
// e4m3_i * 2^(b - 127); byte 255 stands for NaN (its values are 0).  b is the smallest exponent for
// which the group's largest magnitude fits: max|x| <= 448 * 2^(b - 127), clamped at 0; a group of
// zeros has b = 0; a group with a non-finite value has b = 255.  A power of two as scale keeps the
// products x * 2^(127 - b) and e4m3 * 2^(b - 127) exact, so the only rounding is the one to e4m3
// (nearest, ties to even; half a unit in the fourth significant bit).
//
// The 4-bit row: Hkv * D / 2 bytes of e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), then
// the scale bytes as above.  b is the smallest exponent with max|x| <= 7 * 2^(b - 127), clamped to 0 .. 252:
// up to 7 the largest value errs by at most 1 (it becomes 6), half of what the level 8 above would be away, and
// normal groups come out 0.3 dB nearer than with the limit at 6 (19.0 against 18.7).  Up to 252 every value is
// finite in bf16; 253 to 255 stand for NaN (the writer uses 255, with values of 0).
// Order within a head: value 32 g + 4 p + j (p < 8, j < 4) is in byte p * D / 16 + 2 g + j / 2, the low half for even
// j.  So the four values of every group that a lane of the attention's products takes come in one load, and the 16
// dims of a product are of one group: the scales multiply 32-bit sums and the probabilities, not every value.
#pragma once

#include <cuda_fp4.h>
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

constexpr uint32_t kNan4 = 253;             // from here on a scale byte of the 4-bit row stands for NaN

// Scale byte of a 4-bit group whose largest magnitude has the bits `top`: 7 = 1.75 * 2^2, and a mantissa past 1.75 carries.
__device__ __forceinline__ uint32_t scale_byte4(uint32_t top) {
  const int e = int(top + 0x1fffffu >> 23) - 2;
  return top >= 0x7f800000u ? 255u : uint32_t(min(max(e, 0), 252));
}
__device__ __forceinline__ float scale_of4(uint32_t b) { return scale_of(b >= kNan4 ? 255u : b); }

// Four values (the first in the lowest half byte) and back: one conversion per pair.
__device__ __forceinline__ uint32_t f32_e2m1x4(float x0, float x1, float x2, float x3) {
  uint32_t r;                                // (a NaN: any code)
  asm("{\n\t.reg .b8 a, b, z;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "mov.b32 %0, {a, b, a, b};\n\t}"
      : "=r"(r)
      : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
  return r & 0xffffu;
}
__device__ __forceinline__ uint32_t e2m1x2_f16(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(__nv_fp4x2_storage_t(two), __NV_E2M1);
  return uint32_t(h.x) | uint32_t(h.y) << 16;
}
// The eight values of a word, byte i's in r[i], as fp16 (exact).  The compiler is not to look through how the word came about:
// for one put together from two single bytes, upper half zero, nvcc 12.9 made zeros of this.
__device__ __forceinline__ void e2m1x8_f16(uint32_t w, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm("" : "+r"(w));
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
      : "r"(w));
}
__device__ __forceinline__ float2 f16x2_f32(uint32_t h) { return __half22float2(reinterpret_cast<const __half2&>(h)); }

template <bool BF16>
__device__ __forceinline__ uint32_t mul16x2(uint32_t x, uint32_t f) {
  uint32_t r;
  if constexpr (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(f));
  else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(f));
  return r;
}
// The 4-bit cache.  Eight values as 16-bit ones, times the power of two of their scale byte.  fp16 by one conversion
// and one multiplication per pair; bf16 by way of that: the product is exact in fp16 where the scale byte is an ordinary
// one, and goes through 32 bits (half of these five operations off the pipe that converts, which is the busiest here:
// moving fp16's exponent under bf16's by masks and shifts takes four of five on it).
// Whether the scale bytes of a word are ordinary:
template <bool BF16>
__device__ __forceinline__ bool plain_scales4(uint32_t w) {
  return __vcmpgtu4(w, 0x8c8c8c8cu) == 0 && __vcmpgtu4(0x71717171u, w) == 0;    // 113 .. 140
}
__device__ __forceinline__ uint32_t plain_factor4(uint32_t b) { return (b - 112u) * 0x04000400u; }
template <bool BF16>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t f_lo, uint32_t f_hi, uint32_t (&r)[4]) {   // a factor per four values
  e2m1x8_f16(w, r[0], r[1], r[2], r[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = mul16x2<false>(r[i], i < 2 ? f_lo : f_hi);
    if constexpr (BF16) {
      const float2 x = f16x2_f32(r[i]);
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r[i]) : "f"(x.y), "f"(x.x));
    }
  }
}
template <bool BF16>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t f, uint32_t (&r)[4]) { widen4<BF16>(w, f, f, r); }
// ... for any scale byte: two multiplications, of which only the last rounds; fp16 past its range: its largest.  (bf16: the
// exponent and first mantissa bit moved under bf16's exponent read as the value times 2^-112.)
template <bool BF16>
__device__ __forceinline__ void widen4_any(uint32_t w, uint32_t b, uint32_t (&r)[4]) {
  uint32_t f0, f1;
  if constexpr (BF16) {
    const uint32_t e = min(b, 142u);
    f0 = e * 0x00800080u + 0x38003800u;
    f1 = (b - e + 127u) * 0x00800080u;
  } else if (b < 113u) {                       // 2^-14, exact for what comes first, and the rest down to its subnormals
    f0 = 0x04000400u;
    f1 = (b >= 99u ? b - 98u << 10 : (b >= 89u ? 1u << b - 89u : 0u)) * 0x00010001u;
  } else {
    const uint32_t e = min(b, 140u);
    f0 = (e - 112u) * 0x04000400u;
    f1 = (min(b - e, 15u) + 15u) * 0x04000400u;
  }
  if (b >= kNan4) f1 = 0x7fff7fffu;            // NaN
  e2m1x8_f16(w, r[0], r[1], r[2], r[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const uint32_t m = r[i] & 0x7fff7fffu;
      r[i] = (r[i] ^ m) | (m >> 3);
    }
    r[i] = mul16x2<BF16>(mul16x2<BF16>(r[i], f0), f1);
    if constexpr (!BF16) {
      asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(0x7bff7bffu));
      asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(0xfbfffbffu));
    }
  }
}
// Bytes of values of a row, and the row's least length.
__host__ __device__ inline int64_t payload_bytes(int bits, int Hkv, int D) { return int64_t(Hkv) * D * bits / 8; }
__host__ __device__ inline int64_t least_row_bytes(int bits, int Hkv, int D) {
  return payload_bytes(bits, Hkv, D) + int64_t(Hkv) * (D / kQuantGroup);
}
// Value d of head h of a 4-bit row, in 32 bits.
__device__ __forceinline__ float value4(const uint8_t* row, int Hkv, int D, int h, int d) {
  const uint32_t g = uint32_t(d) / 32u, p = uint32_t(d) % 32u / 4u, j = uint32_t(d) & 3u;
  const uint32_t code = row[h * (D / 2) + int(p * (uint32_t(D) / 16u) + 2u * g + j / 2u)] >> (4u * (j & 1u)) & 15u;
  const uint32_t e = code >> 1 & 3u, m = code & 1u;        // 0.5 m, or (1 + 0.5 m) 2^(e - 1)
  const float size = e == 0u ? 0.5f * float(m) : __uint_as_float((126u + e) << 23 | m << 22);
  return (code & 8u ? -size : size) * scale_of4(row[Hkv * (D / 2) + h * (D / kQuantGroup) + int(g)]);
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
