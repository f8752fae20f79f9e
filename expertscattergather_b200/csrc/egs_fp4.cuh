// Rows in 4 bits: blocks of 32 values of one sign, two exponent and one mantissa bit (magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6), two to a byte, the
// first in the lower half, and a power of two for each block, as the byte of a float32's exponent (255: not a number).
#pragma once

#include "egs_internal.cuh"

namespace egs {
namespace {

constexpr int kFp4Block = 32;
__host__ __device__ constexpr int fp4_blocks(int C) { return (C + kFp4Block - 1) / kFp4Block; }

// The scale's byte of a block from its largest magnitude's float32 bits: the smallest power of two s with magnitude <= 7 s.  7 is where rounding to
// nearest still leaves the largest value, 6.  (Relative 2-norm of the error for normal values: 0.1117; never beyond 6: 0.1154; the magnitude's own
// power of two, which leaves up to 8: 0.1148.)
__device__ __forceinline__ uint32_t fp4_scale(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int e = static_cast<int>((top + 0x1fffffu) >> 23) - 2;       // (magnitudes above 1.75 * 2^n go up)
  return e > 0 ? e : 0;
}
// 1 / scale of bytes up to 253, 0 for one that is not a number: such a block holds zeros.
__device__ __forceinline__ float fp4_inverse(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float fp4_power(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}
// A scale as two factors, `low` at most 1 and `high` at least 1 (both NaN of one that is not a number).  A block's sum times `low`, times the other operand's scale,
// times `high` leaves float32's range no earlier than the product itself: sums are multiples of 1/4 up to 1152, so that all but the last factor give
// exact numbers from 2^-129 on, or the last one is 1.  (Times one scale and then the other, rows from 2^118 on gave infinities whatever the weights.)
__device__ __forceinline__ void fp4_factors(float power, float& low, float& high) {
  asm("min.NaN.f32 %0, %2, 0f3F800000;\n\tmax.NaN.f32 %1, %2, 0f3F800000;" : "=f"(low), "=f"(high) : "f"(power));
}

// Eight values to the nearest of 4 bits (ties to an even mantissa, beyond 6: 6).
__device__ __forceinline__ uint32_t fp4_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// One value times the inverse scale.  (0 * infinity in a block of zeros would be a NaN, which 4 bits hold as 6.)
__device__ __forceinline__ float fp4_scaled(float v, float inverse) { return inverse == 0.f ? 0.f : v * inverse; }

// Eight values as twice their 4 bits' in 8-bit integers, four to a word.
__device__ __forceinline__ void fp4_integers(uint32_t w, uint32_t& low, uint32_t& high) {
  constexpr uint32_t p0 = 0x03020100u, p1 = 0x0c080604u, n0 = 0xfdfeff00u, n1 = 0xf4f8fafcu;     // 0 1 2 3 4 6 8 12 and their negatives
  const uint32_t m = w & 0x77777777u, s = (w >> 1) & 0x44444444u;
  low = __byte_perm(__byte_perm(p0, p1, m), __byte_perm(n0, n1, m), 0x3210u + (s & 0xffffu));
  high = __byte_perm(__byte_perm(p0, p1, m >> 16), __byte_perm(n0, n1, m >> 16), 0x3210u + (s >> 16));
}

// What the lowest 4 bits stand for.
__device__ __forceinline__ float fp4_value(uint32_t w) { return __uint_as_float((w & 7u) << 22 | (w & 8u) << 28) * 0x1p126f; }
// Eight values in 4 bits as 16-bit floats, the first in the lowest half.  (Of a word in 32-bit registers: from what the compiler can see to have been bytes, a
// byte's load or a conversion into 4 bits, CUDA 12.9's leaves zeros.)
__device__ __forceinline__ void fp4_halves(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}

struct Block4 {
  uint32_t w[4];
};
// Block c of a row of `C` elements (an even number), zeros behind the row's end.
__device__ __forceinline__ Block4 load_block(const uint8_t* row, int c, int C) {
  Block4 b;
  if ((c + 1) * kFp4Block <= C) {
    const uint4 x = reinterpret_cast<const uint4*>(row)[c];
    b.w[0] = x.x; b.w[1] = x.y; b.w[2] = x.z; b.w[3] = x.w;
  } else {
    const int left = C - c * kFp4Block;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b.w[i] = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (8 * i + 2 * j < left) b.w[i] |= static_cast<uint32_t>(row[c * 16ll + 4 * i + j]) << (8 * j);
    }
  }
  return b;
}

// x / (1 + exp(-x)) as torch's elementary operations form it, bit by bit (the sum is not joined with the exponential's last product).
__device__ __forceinline__ float silu_exact(float x) { return x / __fadd_rn(1.f, expf(-x)); }
// The same within 2^-20, relative, for every x: no branches, so that 32 of them go side by side (65536 rows, 2048 -> 512: 68 us, with silu_exact
// 177, with the fast exponential, which is off by 2^-17 at -70, 60, without an activation 55).  exp(-|x|) is at most 1, so no sum is beyond 2.  In units of 2^-24 the exponential is off by 4, the two
// products and the sum by 1 each, the reciprocal by 2; silu_exact by 6.  From -88.72284 on, the first float beyond the logarithm of the largest, that one's exponential is infinite and its result 0.
__device__ __forceinline__ float silu_near(float x) {
  float t = expf(-fabsf(x)), r;
  if (x <= -88.72284f) t = 0.f;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + t));
  return (x < 0.f ? x * t : x) * r;
}

}  // namespace
}  // namespace egs
