// 8-bit paged cache: number format, conversions and shared host checks.
//
// A pool holds e4m3 codes [L, P, Hkv, bs, D]; every (layer, block, KV head)
// has one fp32 scale for K and one for V, and a stored value is code * scale.
// Scales are powers of two: the smallest 2^k with amax <= 448 * 2^k.  For a
// floating-point code that costs no precision (the mantissa keeps its three
// bits whatever the scale), x / scale is exact, and raising the scale of a block
// that already holds tokens only shifts their exponents: an old code is rounded
// again only where it becomes subnormal (below 2^-6 of the new scale).
#pragma once

#include "common.cuh"

namespace bl {

constexpr int kScaleMinExp = -100;  // below this x / scale could leave fp32's normal range
constexpr int kScaleMaxExp = 119;   // 448 * 2^119 is the largest code value that fits fp32 and bf16

// k of the scale 2^k for a block whose largest finite magnitude is amax:
// amax = 1.m * 2^e <= 448 * 2^k = 1.75 * 2^(k + 8).
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int k = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(k, kScaleMinExp), kScaleMaxExp);
}
__device__ __forceinline__ float exp2_int(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// 1 / 2^k, exact (k within the scales' range)
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// |x| of a finite x, else 0 (NaN compares false).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// two floats -> two e4m3 codes, `lo` in the low byte (nearest even, saturating at 448; NaN -> NaN)
__device__ __forceinline__ uint16_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  return (uint32_t)pack_e4m3x2(a, b) | ((uint32_t)pack_e4m3x2(c, d) << 16);
}

// two e4m3 codes -> packed fp16 pair (exact: every e4m3 value is an fp16 value)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
// the low and the high half of a word of four codes
__device__ __forceinline__ uint32_t e4m3lo_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t e4m3hi_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint16_t v) { return unpack2<__half>(e4m3x2_to_f16x2(v)); }
__device__ __forceinline__ float e4m3_to_float(uint8_t v) { return e4m3x2_to_float2(v).x; }

// code value * scale in the caller's type, saturating at the type's largest
// finite value (only fp16 can get there: 65504 lies below its block's largest code)
template <typename T> __device__ __forceinline__ T dequant_to(float v) { return from_f32<T>(v); }
template <> __device__ __forceinline__ __half dequant_to<__half>(float v) {
  return __float2half_rn(v != v ? v : fminf(fmaxf(v, -65504.f), 65504.f));
}

// Fp16 operands of the matrix instructions.  bf16 holds every code times every scale
// exactly, fp16 does not: 448 * 2^8 is past its range, 2^-9 * 2^-16 below its last bit.
// So for fp16 the values of a row's KV head are taken in units of a power of two, u,
// such that its largest scale becomes 2^7 of them (codes up to 57344): exact for
// the blocks whose scale is within 2^22 of the largest, and to 2^-25 u, less than
// 2^-40 of the largest code's value, for the others.  The products take u back in fp32.
__device__ __forceinline__ float half_unit(float largest_scale) {
  const uint32_t e = __float_as_uint(largest_scale) >> 23;  // (0: no block; 255: no scale that an append leaves)
  return e > 7 && e < 255 ? __uint_as_float((e - 7) << 23) : 1.f;
}
// code * scale of two codes, packed
template <typename T> __device__ __forceinline__ uint32_t dequant2(float2 x, float s) {
  return pack2<T>(x.x * s, x.y * s);
}
// eight codes times scale, as 16-bit values
template <typename T> __device__ __forceinline__ uint4 dequant8(uint2 c, float s) {
  return make_uint4(dequant2<T>(unpack2<__half>(e4m3lo_to_f16x2(c.x)), s), dequant2<T>(unpack2<__half>(e4m3hi_to_f16x2(c.x)), s),
                    dequant2<T>(unpack2<__half>(e4m3lo_to_f16x2(c.y)), s), dequant2<T>(unpack2<__half>(e4m3hi_to_f16x2(c.y)), s));
}

// Validates an 8-bit layer: the shared checks plus the scale tables.
inline int check_fp8_layer(const bl_fp8_layer& l, const char* who) {
  const int rc = check_paged_layer(l.kv, who);
  if (rc) return rc;
  BL_CHECK_ARG(l.k_scale && l.v_scale, "%s: scale pointers must be non-null", who);
  BL_CHECK_ARG(((uintptr_t)l.kv.k_pool & 15) == 0 && ((uintptr_t)l.kv.v_pool & 15) == 0,
               "%s: pools must be 16-byte aligned", who);
  BL_CHECK_ARG(l.kv.head_dim <= 256, "%s: head_dim > 256 is not supported", who);
  BL_CHECK_ARG(l.kv.num_kv_heads <= 65535, "%s: too many KV heads", who);
  BL_CHECK_ARG(l.kv.block_size <= 65536, "%s: block_size > 65536 is not supported", who);
  return BL_OK;
}

}  // namespace bl
