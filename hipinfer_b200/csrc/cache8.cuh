// A paged cache in 8 bits: codes [page][kv head][page_size][D], int8 or e4m3, and one float32 scale for each block of 16 places of
// a page and head, [page][kv head][ceil(page_size / 16)]; a place's numbers are code * scale. Keys and values have their own.
#pragma once
#include "common.cuh"

#include <cuda_fp8.h>

enum { HB_I8 = 2, HB_E4M3 = 3 };                // codes of the code types, beside HB_F32 and HB_BF16
constexpr int C8_BLOCK = 16;                    // places that share a scale
constexpr float C8_LEAST = 1e-30f;              // below it a block's largest number counts as this: no scale is 0 or denormal

__host__ __device__ constexpr int c8_blocks(int page_size) { return (page_size + C8_BLOCK - 1) / C8_BLOCK; }

// A code type: its largest number, code to number (four of them from four bytes), and number (already within +- the largest) to the nearest code, ties to the even one; four of them
// to four bytes.
struct C8Int8 {
  static constexpr float MOST = 127.f;
  static __device__ __forceinline__ float value(uint8_t c) { return (float)(int8_t)c; }
  // (with the sign bit turned a byte u is code + 128, and 0x4b000000 | u is 2^23 + u)
  static __device__ __forceinline__ void values4(uint32_t w, float* x) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 + i)) - 8388736.f;
  }
  // (1.5 x 2^23 + x has x's nearest integer in its last bits, ties to even; conversions to integers run at an eighth of an addition's rate)
  static __device__ __forceinline__ uint32_t code4(const float* x) {
    const uint32_t a = __float_as_uint(__fadd_rn(x[0], 12582912.f)), b = __float_as_uint(__fadd_rn(x[1], 12582912.f));
    const uint32_t c = __float_as_uint(__fadd_rn(x[2], 12582912.f)), d = __float_as_uint(__fadd_rn(x[3], 12582912.f));
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  }
  static __device__ __forceinline__ uint8_t code(float x) { return (uint8_t)__float_as_uint(__fadd_rn(x, 12582912.f)); }
};
struct C8E4m3 {
  static constexpr float MOST = 448.f;
  static __device__ __forceinline__ float value(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
  }
  static __device__ __forceinline__ void values4(uint32_t w, float* x) {
    const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3)), b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
    const float2 p = __half22float2(a), q = __half22float2(b);
    x[0] = p.x, x[1] = p.y, x[2] = q.x, x[3] = q.y;
  }
  static __device__ __forceinline__ uint32_t code4(const float* x) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3) << 16;
  }
  static __device__ __forceinline__ uint8_t code(float x) { return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }
};

#define C8_DISPATCH(ct, NAME, ...)                                  \
  do {                                                              \
    if ((ct) == HB_I8) { using CT = C8Int8; __VA_ARGS__; }          \
    else if ((ct) == HB_E4M3) { using CT = C8E4m3; __VA_ARGS__; }   \
    else HB_FAIL("%s: unknown code type %d", NAME, (int)(ct));      \
  } while (0)
