// Codes of the 8-bit key/value cache: q8 (signed whole numbers) and e4m3, one f32 scale per row.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace dyn {

__device__ __forceinline__ float kv_float(float x) { return x; }
__device__ __forceinline__ float kv_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float kv_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void kv_store(float x, float* y) { *y = x; }
__device__ __forceinline__ void kv_store(float x, __half* y) { *y = __float2half_rn(x); }
__device__ __forceinline__ void kv_store(float x, __nv_bfloat16* y) { *y = __float2bfloat16_rn(x); }

// The row's scale and the factor its entries are multiplied with, from the bits of its largest magnitude.
template <bool E4M3>
__device__ __forceinline__ void kv_scale(uint32_t top, float* scale, float* inv) {
  if (top >= 0x7f800000u) {
    *scale = __uint_as_float(0x7fc00000u), *inv = 0.f;
  } else if (top < (27u << 23)) {  // below 2^-100
    *scale = 0.f, *inv = 0.f;
  } else if (E4M3) {
    // top = 1.m * 2^e: 448 = 1.75 * 2^8, so 2^(e - 8), or the next one where 1.m is above 1.75
    const uint32_t e = (top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    *scale = __uint_as_float(e << 23), *inv = __uint_as_float((254u - e) << 23);
  } else {
    *scale = __fdiv_rn(__uint_as_float(top), 127.f), *inv = __fdiv_rn(127.f, __uint_as_float(top));
  }
}

template <bool E4M3>
__device__ __forceinline__ uint2 kv_encode8(const float (&v)[8], float inv) {
  uint32_t w[2] = {};
  if (inv == 0.f) return make_uint2(0, 0);  // 0 * infinity has no place in the codes
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    uint32_t pair;
    if (E4M3) {
      pair = __nv_cvt_float2_to_fp8x2(make_float2(v[i] * inv, v[i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    } else {
      // the sum's last mantissa bits are the whole number, in two's complement
      const uint32_t p = __float_as_uint(__fmaf_rn(v[i], inv, 12582912.f)), q = __float_as_uint(__fmaf_rn(v[i + 1], inv, 12582912.f));
      pair = (p & 0xffu) | ((q & 0xffu) << 8);
    }
    w[i / 4] |= pair << (i % 4 * 8);
  }
  return make_uint2(w[0], w[1]);
}

// Two q8 codes with 128 added, one in each half's lower byte: 0x6400 | u is the f16 number 1024 + u.
__device__ __forceinline__ uint32_t kv_q8_to_half2(uint32_t bytes) {
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&bytes), __half2half2(__ushort_as_half(0x6480)));  // 1152
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool E4M3>
__device__ __forceinline__ void kv_decode8(uint2 raw, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t byte = ((i < 4 ? raw.x : raw.y) >> (i % 4 * 8)) & 0xffu;
    const float code = E4M3 ? __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)))
                            : (float)(int)(signed char)byte;
    v[i] = code * scale;
  }
}

}  // namespace dyn
