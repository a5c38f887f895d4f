// The 8-bit row format of the K/V pool (include/mac_b200_chunk.h): e4m3 codes and one
// power-of-two scale per (token, KV head) row, kept as its biased exponent.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace mac_b200 {

constexpr int kKv8MinExp = 3;     // 2^-124: the smallest code (2^-9) times it is the smallest bf16
constexpr int kKv8MaxExp = 247;   // 2^120: rows that reach 1.75 * 2^127
constexpr int kKv8NanExp = 255;   // row with an infinity or a NaN

// Exponent byte of a row from the bits of max|x| (finite): the smallest s = 2^(e-127) with
// max|x| / s <= 448 = 1.75 * 2^8, so one binade up where the mantissa exceeds 1.75.
__device__ __forceinline__ int kv8_exp_of(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kKv8MinExp ? kKv8MinExp : e;
}
// 2^(127-e), e in [3, 247]: a normal fp32 number, so x * it rounds nothing unless it underflows
__device__ __forceinline__ float kv8_inverse(int e) {
  return __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}
__device__ __forceinline__ float kv8_scale(int e) {
  if (e == kKv8NanExp) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(e == 0 ? 0x00400000u : static_cast<uint32_t>(e) << 23);
}
// four values -> four codes, lowest byte first
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
// two codes (low 16 bits) -> their values; every e4m3 number is an fp16 number
__device__ __forceinline__ float2 kv8_unpack2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// 32 bytes: one store of a whole sector where the address allows it, since half a sector costs the memory
// system as much (measured in turn: chunk attention, 8 prompts of 1500-2048 in a band of 1024, 5 % less
// than with 16-byte stores, and 5 % less again with none; 100000 rows read back from the 8-bit pool 101 us
// instead of 109).
__device__ __forceinline__ void store32(uint4* dst, const uint32_t (&w)[8], bool aligned32) {
  if (aligned32) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

}  // namespace mac_b200
