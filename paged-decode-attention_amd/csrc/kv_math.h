// The stored forms of a KV cache as fp16 operands, and the loads of its pages:
// shared by the attention kernels of this library. (int8: the decode rounds the
// product with the scale to fp16, the prompt kernels take the values as they are and
// their scales in fp32.)
#ifndef PA_KV_MATH_H_
#define PA_KV_MATH_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pagedattn.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kInt8Sign = 0x80808080u;      // int8 x -> x + 128 in every byte
constexpr float kInt8Unit = 16777216.0f;      // 2^24: int8 V operands are (x + 128) * 2^-24
// Buffer resource word 3 for raw (stride 0) byte buffers on gfx9, and the
// non-temporal cache policy of a buffer load (bit 1 = nt).
constexpr int kRsrcWord3 = 0x00020000;
constexpr int kLoadNT = 2;

// v_perm_b32: byte k of the result is byte sel[k] of the 8 bytes {hi, lo}
// (codes 0-3 pick `lo`, 4-7 pick `hi`, 0x0c gives 0x00).
__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}

__device__ __forceinline__ f16x8 as_f16x8(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  u32x4 u = {w0, w1, w2, w3};
  return __builtin_bit_cast(f16x8, u);
}

// Two bf16 values (one dword) -> two fp16, each rounded to nearest even.
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t w) {
  const f16x2 h = {(_Float16)__uint_as_float(w << 16), (_Float16)__uint_as_float(w & 0xffff0000u)};
  return __builtin_bit_cast(uint32_t, h);
}

__device__ __forceinline__ f16x8 bf16x8_to_f16x8(u32x4 w) {
  return as_f16x8(bf16x2_to_f16x2(w.x), bf16x2_to_f16x2(w.y), bf16x2_to_f16x2(w.z),
                  bf16x2_to_f16x2(w.w));
}

// fp32 -> bf16 bits, round to nearest even (NaN stays NaN).
__device__ __forceinline__ uint32_t f32_to_bf16_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// Selector placing byte i of `lo` and byte j of `hi` into the two halves of a
// dword: as the high byte (fp8 e5m2 -> fp16) or the low byte (int8 with its
// sign bit flipped -> the fp16 denormal (x + 128) * 2^-24).
template <int KV>
__device__ __forceinline__ constexpr uint32_t pair_sel(uint32_t i, uint32_t j) {
  if constexpr (KV == PA_KV_INT8) {
    return i | (0x0cu << 8) | ((4u + j) << 16) | (0x0cu << 24);
  } else {
    return 0x0cu | (i << 8) | (0x0cu << 16) | ((4u + j) << 24);
  }
}

// Two stored bytes -> two fp16 bit patterns: one v_perm (int8 sign bits are
// flipped on the words before it).
template <int KV>
__device__ __forceinline__ uint32_t bytes_to_halves(uint32_t hi, uint32_t lo, uint32_t sel) {
  return perm(hi, lo, sel);
}

// Two fp32 values -> an fp16 pair, each rounded to nearest even
// (v_cvt_pk_f16_f32). The empty asm statements hide where a and b come from,
// so the compiler converts the fp32 values as they are instead of folding
// the conversion into the fma that produced them (v_fma_mixlo/hi_f16, which
// runs at a third of the rate of ordinary VALU ops when waves share a SIMD).
// They emit no instruction: an instruction written in asm escapes the
// compiler's hazard checks, and an MFMA reading its result one instruction
// later read a stale register.
__device__ __forceinline__ uint32_t cvt_pk_f16(float a, float b) {
  asm("" : "+v"(a));
  asm("" : "+v"(b));
  const f16x2 h = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, h);
}

// int8 -> fp16(x * s), the reference's dequantised value (cache.py:51-62;
// triton_decode.py:145-149: the fp32 product rounded to fp16), for a pair of
// stored bytes whose sign bits are already flipped (b ^ 0x80 = x + 128).
//   fp16 scales: the byte under the exponent byte 0x64 is the fp16 value
//     1024 + (x + 128); minus 1152 it is x, exactly, and one fp16 multiply
//     by s rounds the exact product x * s once (an 8-bit x times an 11-bit s
//     is exact in fp32, so this equals the reference's two roundings).
//     `lo` holds both bytes (positions i, j); 3 packed ops per pair.
//   fp32 scales: the byte as the fp16 denormal (x + 128) * 2^-24 (exact), one
//     fma per element in fp32 with s * 2^24 and -128 * s gives fp32(x * s),
//     then a round to fp16: the reference's fp32 product and fp16 cast.
constexpr uint32_t kF16Exp1024 = 0x64646464u;  // exponent byte of 1024 in every byte

__device__ __forceinline__ uint32_t i8pair_fp16_scale(uint32_t lo, uint32_t i, uint32_t j, uint32_t s2) {
  const uint32_t h = perm(kF16Exp1024, lo, i | (4u << 8) | (j << 16) | (4u << 24));
  const f16x2 x = __builtin_bit_cast(f16x2, h) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f};
  return __builtin_bit_cast(uint32_t, x * __builtin_bit_cast(f16x2, s2));
}

__device__ __forceinline__ uint32_t i8pair_fp32_scale(uint32_t den, float s0_24, float c0, float s1_24,
                                                      float c1) {
  const f16x2 u2 = __builtin_bit_cast(f16x2, den);
  return cvt_pk_f16(__builtin_fmaf((float)u2[0], s0_24, c0), __builtin_fmaf((float)u2[1], s1_24, c1));
}

// A raw buffer over the `bytes` bytes from `base` on: a load at a per-lane
// offset at or past `bytes` returns zeros (the range check of raw buffers).
// bytes = -1 (2^32 - 1) leaves every offset used here in range.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rsrc(const uint8_t *base, int bytes = -1) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), (short)0, bytes, kRsrcWord3);
}

// Block tables and lengths are read-only for a whole launch. Reading them
// through the constant address space lets the compiler use scalar loads for
// the wave-uniform reads even in kernels that store inside their tile loop;
// a scalar load's wait (lgkmcnt) never holds back the K/V loads in flight,
// where a vector load's (vmcnt) would wait for them.
typedef __attribute__((address_space(4))) const int32_t ro_i32;
__device__ __forceinline__ const ro_i32 *ro(const int32_t *ptr) { return (const ro_i32 *)ptr; }

}  // namespace

#endif  // PA_KV_MATH_H_
