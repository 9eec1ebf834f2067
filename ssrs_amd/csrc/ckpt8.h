// The 8-bit activation checkpoint (gfx950 device helpers shared by ckpt8.hip and lora_pool.hip).
//
// A row of C elements is held as blocks of 32 consecutive elements (the last block of a row may be shorter). With amax the largest
// magnitude of a block, e is the smallest integer in [-126, 121] with amax <= 127 * 2^e (121 if there is none: the top half binade of
// fp32 saturates), an element is the int8 code rint(x * 2^-e) (ties to even, clamped to +-127) and stands for code * 2^e. A block keeps
// the byte e + 127; byte 255 marks a block with an infinity or NaN in it, all of whose elements stand for NaN (an overflow must reach
// the gradients, an 8-bit code cannot carry it).
//
// Why a power of two and not amax / 127 itself: x * 2^-e is exact, so the code depends on no rounding but its own (every
// implementation finds the same codes), the scale is one byte, and code * 2^e has at most 7 significant bits: EXACT in bf16, so the
// MFMA kernels that read a checkpoint multiply exactly what it stands for. Price: the step lies between amax/127 and amax/63.5.
#pragma once
#include "common.h"

#define CKPT8_BLOCK 32

__device__ __forceinline__ unsigned int ckpt8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// exponent byte from the largest magnitude's bits (as integers they are ordered, infinities and NaN above all numbers).
// 127 = 1.984375 * 2^6: a mantissa above 0x7e0000 carries into the exponent field when 0x1ffff is added.
__device__ __forceinline__ unsigned int ckpt8_exp_byte(unsigned int amax_bits) {
  int e = (int)((amax_bits + 0x1ffffu) >> 23) - 6;
  e = e < 1 ? 1 : (e > 248 ? 248 : e);
  return amax_bits >= 0x7f800000u ? 255u : (unsigned int)e;
}
__device__ __forceinline__ float ckpt8_step(unsigned int byte) {      // 2^e, NaN for byte 255
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}
__device__ __forceinline__ float ckpt8_inv_step(unsigned int byte) {  // 2^-e, exact; 0 for byte 255 (codes 0)
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
// code in the low byte: clamp, then round to nearest even by adding 1.5 * 2^23
__device__ __forceinline__ unsigned int ckpt8_code(float x, float inv) {
  const float t = __builtin_amdgcn_fmed3f(x * inv, -127.f, 127.f);
  return __float_as_uint(t + 12582912.f) & 0xffu;
}
__device__ __forceinline__ unsigned int ckpt8_code4(float a, float b, float c, float d, float inv) {
  const unsigned int ua = __float_as_uint(__builtin_amdgcn_fmed3f(a * inv, -127.f, 127.f) + 12582912.f);
  const unsigned int ub = __float_as_uint(__builtin_amdgcn_fmed3f(b * inv, -127.f, 127.f) + 12582912.f);
  const unsigned int uc = __float_as_uint(__builtin_amdgcn_fmed3f(c * inv, -127.f, 127.f) + 12582912.f);
  const unsigned int ud = __float_as_uint(__builtin_amdgcn_fmed3f(d * inv, -127.f, 127.f) + 12582912.f);
  const unsigned int lo = __builtin_amdgcn_perm(ub, ua, 0x0c0c0400u);      // bytes: ua.0, ub.0, 0, 0
  const unsigned int hi = __builtin_amdgcn_perm(ud, uc, 0x04000c0cu);      // bytes: 0, 0, uc.0, ud.0
  return lo | hi;
}
__device__ __forceinline__ float ckpt8_value(unsigned int word, int byte, float step) {
  return (float)(signed char)(word >> (8 * byte)) * step;
}
