// Storage of the 4-bit key/value cache, shared by the kernels that write and read it.
//
// A cache is uint8 [pages, kv heads, page_size / 16 records].  A record holds 16 tokens of one kv head in 18 D bytes: key codes (8 D),
// key scales (D), value codes (8 D), value scales (D), E2M1 two to a byte (the even channel low) and one E4M3 scale per 16 channels.  What a
// warp of the attention kernel's mma.sync fragments needs lies side by side, so that each of its loads is 512 (D=128) or 256
// contiguous bytes without an exchange or a bank conflict; lane = 4 n + c of the fragments:
//   key codes     token n or n + 8, channels c D/4 ... : rows of D/2 bytes, in token order
//   key scales    byte (4 n + c) D/32 + (token >> 3) D/64 + (block & (D/64 - 1)); block c D/64 ... : D/32 bytes per lane
//   value codes   tokens 2 c, 2 c + 1 (+ 8), channels n D/8 ... : byte (token >> 3) 4 D + n D/2 + c D/8 + (token & 1) D/16
//   value scales  block b, tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9: byte 16 b + 4 c + 2 (token >> 3) + (token & 1)
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace sage3 {

template <int D>
struct KvRecord {
  static constexpr int kKeyScales = 8 * D, kValues = 9 * D, kValueScales = 17 * D, kBytes = 18 * D;
  // byte of channel `ch` (even) of token t in 0 ... 15, and of the scale of 16-channel block b
  static __device__ __forceinline__ int key(int t, int ch) { return t * (D / 2) + ch / 2; }
  static __device__ __forceinline__ int key_scale(int t, int b) {
    constexpr int S = D / 64;
    return kKeyScales + (4 * (t & 7) + b / S) * (2 * S) + (t >> 3) * S + b % S;
  }
  static __device__ __forceinline__ int value(int t, int ch) {
    return kValues + (t >> 3) * (4 * D) + ch / (D / 8) * (D / 2) + ((t >> 1) & 3) * (D / 8) + (t & 1) * (D / 16) + ch % (D / 8) / 2;
  }
  static __device__ __forceinline__ int value_scale(int t, int b) {
    return kValueScales + 16 * b + 4 * ((t >> 1) & 3) + 2 * (t >> 3) + (t & 1);
  }
};

// 8 codes (a word) -> 4 pairs of fp16
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\ncvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// two scales (the low half word) -> a pair of fp16, exact: E4M3 is a subset of fp16
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t w) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)w));
  return h;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float2 f16x2_to_f32(uint32_t h) { return __half22float2(*reinterpret_cast<__half2*>(&h)); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}

}  // namespace sage3
