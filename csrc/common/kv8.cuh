// The 8-bit key / value cache: uint8 [blocks][2][kv_head] pages, a page = block_size rows of D e4m3 codes, then block_size fp32
// scales.  A row (one token's key or value of one head) is code * scale with
//     scale = 2^e, e the smallest of -15 .. 7 with max |x| <= 448 * 2^e (7 if there is none),   code = e4m3(x / scale), saturating.
// Powers of two cost no accuracy (codes are floating point: a scale moves their range, not their steps) and make every stored
// value an exact fp16 and bf16 number: the largest is 448 * 2^7 = 57344, the smallest 2^-9 * 2^-15.
// A token whose key or value row of a head holds a NaN has NaN for both scales of that head, and codes of zero: attention finds
// out from the key alone, and no NaN sits among the codes, where a product with a weight of zero would spread it to other rows.
#pragma once
#include <cuda_fp8.h>

#include "utils.cuh"

namespace b200 {

constexpr float kKv8Max = 448.f;

struct Kv8Cache {
  uint8_t* base;
  int64_t num_blocks;
  int Hkv, block_size, D;
  __host__ __device__ int64_t page_bytes() const { return (int64_t)block_size * (D + 4); }
  __device__ __forceinline__ uint8_t* page(int64_t blk, int which, int h) const {
    return base + ((blk * 2 + which) * Hkv + h) * page_bytes();
  }
  __device__ __forceinline__ uint8_t* codes(uint8_t* page, int off) const { return page + (int64_t)off * D; }
  __device__ __forceinline__ float* scale(uint8_t* page, int off) const {
    return reinterpret_cast<float*>(page + (int64_t)block_size * D) + off;
  }
};

__device__ __forceinline__ bool is_nan_bits(float v) { return (__float_as_uint(v) & 0x7fffffffu) > 0x7f800000u; }

// scale of a row whose largest magnitude is amax (not a NaN; infinity saturates)
__device__ __forceinline__ float kv8_scale(float amax) {
  const float s = pow2_ceil(__fdiv_rn(fminf(amax, kKv8Max * 128.f), kKv8Max));
  return fminf(fmaxf(s, 1.f / 32768.f), 128.f);
}
// exact reciprocal of a power of two
__device__ __forceinline__ float pow2_inv(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// eight scaled values -> eight codes
__device__ __forceinline__ uint2 kv8_pack8(const float (&v)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | hi << 16;
  }
  return make_uint2(w[0], w[1]);
}
// two codes -> two fp16 numbers (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}
// and back, rounded; e5m2 numbers are the upper bytes of fp16 numbers
__device__ __forceinline__ uint16_t f16x2_to_e4m3x2(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&v)));
  return r;
}
__device__ __forceinline__ uint16_t f16x2_to_e5m2x2(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&v)));
  return r;
}
__device__ __forceinline__ uint32_t e5m2x2_to_f16x2(uint16_t v) { return __byte_perm(v, 0, 0x1404); }
__device__ __forceinline__ float2 e4m3x2_to_float2(uint16_t c) {
  const uint32_t r = e4m3x2_to_f16x2(c);
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}

}  // namespace b200
