// 8-bit activation checkpoints: the storage format and its device-side conversions, shared by the
// kernels that write and read it (ckpt8.cu, glu.cu, affine_bwd.cu).
//
// A row of `cols` values is cut into groups of 32 consecutive ones. Per group one byte
//   b = max(7, biased fp32 exponent of the largest magnitude),
// fixes the step delta = 2^(b - 133), and every value is kept as the int8 code
//   k = clamp(round_half_even(x / delta), -127, 127);  it stands for k * delta.
// The largest magnitude lies in [64, 128) steps, so |x - k*delta| <= delta / 2, except in the last
// half step of the range (above 127.5 steps), where the clamp makes it less than one delta. The
// step is a power of two on purpose: the scaling, the rounding and k * delta (seven significant
// bits, never below the normal range) are exact in fp32 and in bfloat16, so a checkpoint has one
// right value, bit for bit, and the weight gradient can feed it to the tensor cores unrounded.
// A group with a value that is not finite has b = 255 and codes 0, and stands for NaN throughout.
// Memory: codes [rows, 32 * groups], groups = ceil(cols / 32), codes past `cols` are 0, so every row
// of codes starts on a 32-byte boundary whatever `cols`; exponents [rows, groups].
#pragma once

#include <cuda_bf16.h>

#include "dwbnq_device.cuh"

namespace dwbnq {

template <> struct Elem<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
};

constexpr int kCkGroup = 32;
constexpr unsigned int kCkMinExp = 7;    // delta and 1 / delta stay normal fp32 numbers
constexpr unsigned int kCkNonFinite = 255;

// Exponent byte from the largest magnitude's bit pattern (NaN and infinity have the exponent 255).
__device__ __forceinline__ unsigned int ck_exponent(unsigned int abs_bits) {
  const unsigned int b = abs_bits >> 23;
  return b < kCkMinExp ? kCkMinExp : b;
}
// 1 / delta; 0 for a group that is not finite (then every code comes out as 0).
__device__ __forceinline__ float ck_inv_step(unsigned int b) {
  return b == kCkNonFinite ? 0.0f : __uint_as_float((260u - b) << 23);
}
// delta; NaN for a group that is not finite.
__device__ __forceinline__ float ck_step(unsigned int b) {
  return b == kCkNonFinite ? __uint_as_float(0x7fc00000u) : __uint_as_float((b - 6u) << 23);
}
__device__ __forceinline__ int ck_code(float x, float inv) {
  // fminf / fmaxf drop the NaN that a value that is not finite leaves (0 * inf): code 0 by the last select
  const float t = fminf(fmaxf(__fmul_rn(x, inv), -127.0f), 127.0f);
  return inv == 0.0f ? 0 : __float2int_rn(t);
}

}  // namespace dwbnq
