// What a page of the paged K/V cache holds, and the conversions between it and 16-bit or fp32 values.
//
// 16-bit cache: a page is [block_size][kv_heads][head_dim] of the model's type.
// 8-bit cache:  a page is the codes [block_size][kv_heads][head_dim], one byte each, and behind them the
// fp32 scales [block_size][kv_heads], padded to a multiple of 16 bytes.  A value is code * scale.  Codes and
// scales form ONE run of bytes, so the swap and migration kernels, which know a page only as bytes, carry
// an 8-bit page with its scales and need no second call.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "common.cuh"

namespace hfk {

constexpr int kFmtRaw = HFK_KV_RAW, kFmtE4m3 = HFK_KV_E4M3, kFmtInt8 = HFK_KV_INT8;

// Largest code, and the least scale (the smallest normal fp32 number: a row of zeros gets it, and its
// reciprocal is finite).
template <int kFmt>
__device__ __forceinline__ constexpr float top_code() { return kFmt == kFmtE4m3 ? 448.f : 127.f; }
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126

// n / d and n % d for 0 <= n < 2^31 with one multiplication: mul = ceil(2^(31+l) / d), l = ceil(log2 d).
// mul * d exceeds 2^(31+l) by less than d <= 2^l, so the quotient is exact for n < 2^31.
struct FastDiv {
  uint32_t d, mul, shift;
  __host__ static FastDiv make(uint32_t d) {
    FastDiv f;
    f.d = d;
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    f.mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
    f.shift = l == 0 ? 0 : l - 1;
    return f;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};

// ---- 16-bit types ---------------------------------------------------------------------------------------
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
};
template <> struct Pair<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
};

// ---- codes to fp32 ----------------------------------------------------------------------------------------
// Four codes of a word.  e4m3 through fp16, which holds every e4m3 number; int8: code ^ 0x80 is code + 128,
// placed in the low mantissa byte of 2^23, and 2^23 + 128 is subtracted again (exact).
template <int kFmt>
__device__ __forceinline__ void codes_to_float(uint32_t w, float *x) {
  if (kFmt == kFmtE4m3) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
      const float2 f = __half22float2(__half2(r));
      x[2 * h] = f.x;
      x[2 * h + 1] = f.y;
    }
  } else {
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + i)) - 8388736.f;
  }
}

// Four fp32 numbers within the format's range (or NaN) to codes, ties to even.  int8: adding 1.5 * 2^23
// leaves the rounded integer in the low byte.
template <int kFmt>
__device__ __forceinline__ uint32_t float_to_codes(float a, float b, float c, float d) {
  if (kFmt == kFmtE4m3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  constexpr float kMagic = 12582912.f;
  const uint32_t ia = __float_as_uint(a + kMagic), ib = __float_as_uint(b + kMagic);
  const uint32_t ic = __float_as_uint(c + kMagic), id = __float_as_uint(d + kMagic);
  return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

}  // namespace hfk
