// Device helpers of the 8-bit KV cache: e4m3 codes with one f32 scale for each
// (block, KV head), value = code * scale.
//
// Codes widen to f16 exactly (e4m3 is 4 significant bits over 2^-9 .. 448, all
// inside f16), so the attention kernels multiply f16 x f16 into f32: K and V
// enter without rounding, the softmax weights keep 11 bits instead of bf16's 8,
// and q (bf16) is scaled by a power of two per head row so that it fits f16
// exactly except for elements more than 2^29 below the row's largest.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace muk {

constexpr int kKvBlock = 16;        // tokens of a paged block (only size)
constexpr float kE4m3Max = 448.f;
// Scales lie in [2^-60, 2^60] (or are NaN, see below): the appends write powers
// of two in that range, and the attention kernels clamp to it, which keeps the
// products of two scales and a softmax weight inside f32.
constexpr int kScaleExpMin = -60;
constexpr int kScaleExpMax = 60;

// 2^e, exact, e in [-126, 127].
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// Smallest e with amax <= 448 * 2^e, held to the scale range; amax is given by
// its bits (finite, >= 0).  448 = 0.875 * 2^9, so with amax = m * 2^x, m in
// [0.5, 1), that is x - 9, plus one where m > 0.875.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  const int x = (int)(amax_bits >> 23) - 126;
  int e = x - 9 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < kScaleExpMin ? kScaleExpMin : e;
  return e > kScaleExpMax ? kScaleExpMax : e;
}

// A scale as the attention kernels use it: clamped to the range, NaN kept (a
// block that holds a non-finite value reads as NaN).
__device__ __forceinline__ float clamp_scale(float s) {
  s = s < pow2i(kScaleExpMin) ? pow2i(kScaleExpMin) : s;
  return s > pow2i(kScaleExpMax) ? pow2i(kScaleExpMax) : s;
}

// Two e4m3 codes (low 16 bits of v) -> f16x2, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(r) : "r"(v));
  return r;
}
// Four codes -> two f16x2.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t v, uint32_t& a, uint32_t& b) {
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
      : "=r"(a), "=r"(b)
      : "r"(v));
}
// Four f32 -> four codes, rounded to nearest even, saturated at +-448.
__device__ __forceinline__ uint32_t f32x4_to_e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\nmov.b32 %0, {lo, hi};\n}\n"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack_f16x2(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

// The factor 2^f that brings a row whose largest |x| has these bits into
// [2^to, 2^(to + 1)) (f held to what an f32 can scale by; zero and non-finite rows: 1),
// and its inverse.
__device__ __forceinline__ void row_factor(uint32_t max_bits, int to, float& up, float& down) {
  const int x = (int)(max_bits >> 23);           // biased exponent
  int f = (x == 0 || x == 255) ? 0 : to - (x - 127);
  f = f > 126 ? 126 : (f < -126 ? -126 : f);
  up = pow2i(f);
  down = pow2i(-f);
}

// m16n8k16, f16 x f16 -> f32.
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8x8 matrix of 16-bit elements held two to a lane.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src));
}
__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

}  // namespace muk
