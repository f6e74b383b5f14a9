// The 4-bit group format shared by the decode linears' weights (linear4.cu) and the key/value cache
// (kv4.cu).
//
// A group of consecutive values has one scale s and codes c = round(x / s), ties to even, |c| <= 7,
// stored as c + 8.  s is the smallest number with FIVE significant bits that is >= amax / 7 (amax the
// group's largest magnitude), so no code saturates and, with three significant bits of c, s * c has at
// most eight: it is a bf16 number exactly.  A dequantised operand of a bf16 tensor-core product
// therefore carries no rounding, at the price of a step at most 1/16 wider than amax / 7.
//
// Groups with amax < 2^-110 are stored as zeros (s = 0), magnitudes above 2^120 saturate there (16 s
// and 24 s, the dequantiser's factors, stay finite), and a group holding an infinity or a NaN gets
// s = NaN: every value of it reads back as NaN.
//
// Both roundings are decided exactly.  7 s needs eight bits, so 7 s >= amax is an exact comparison that
// corrects amax / 7 for its own rounding; and r = 2 x - 2 c s is exact in the type of x for the nearest
// codes (c s needs eight bits, and r's magnitude is at most about 2 s, near the lowest bit of both), so
// comparing it with s finds the nearest code and its ties whatever x * (1 / s) rounded to.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace nsa {

constexpr int kKvGroup = 32;   // values per scale of the cache, along the head dim

__device__ __forceinline__ float q4_scale(float amax) {
  if (amax < 0x1p-110f) return 0.f;
  if (!(amax <= 3.4028235e38f)) return __uint_as_float(0x7FC00000u);
  amax = fminf(amax, 0x1p120f);
  const uint32_t lo = __float_as_uint(__fdiv_rn(amax, 7.f)) & 0xFFF80000u;   // four bits after the leading one
  return 7.f * __uint_as_float(lo) >= amax ? __uint_as_float(lo) : __uint_as_float(lo + 0x00080000u);
}

__device__ __forceinline__ float q4_scale(double amax) {
  if (amax < 0x1p-110) return 0.f;
  if (!(amax <= 1.7976931348623157e308)) return __uint_as_float(0x7FC00000u);
  amax = fmin(amax, 0x1p120);
  const unsigned long long lo = (unsigned long long)__double_as_longlong(amax / 7.0) & 0xFFFF000000000000ull;
  const double s = __longlong_as_double((long long)lo);
  return (float)(7.0 * s >= amax ? s : __longlong_as_double((long long)(lo + 0x0001000000000000ull)));
}

// Stored code (c + 8) of x for scale s > 0; inv is about 1 / s.
__device__ __forceinline__ uint32_t q4_code(float x, float s, float inv) {
  x = fminf(fmaxf(x, -0x1p120f), 0x1p120f);
  float c = rintf(x * inv);
  const float r = fmaf(-2.f * c, s, 2.f * x);
  const bool odd = ((int)c & 1) != 0;
  if (r > s || (r == s && odd)) c += 1.f;
  else if (r < -s || (r == -s && odd)) c -= 1.f;
  return (uint32_t)((int)fminf(fmaxf(c, -7.f), 7.f) + 8);
}

__device__ __forceinline__ uint32_t q4_code(double x, double s, double inv) {
  x = fmin(fmax(x, -0x1p120), 0x1p120);
  double c = rint(x * inv);
  const double r = fma(-2.0 * c, s, 2.0 * x);
  const bool odd = ((int)c & 1) != 0;
  if (r > s || (r == s && odd)) c += 1.0;
  else if (r < -s || (r == -s && odd)) c -= 1.0;
  return (uint32_t)((int)fmin(fmax(c, -7.0), 7.0) + 8);
}

// Largest magnitude of two, keeping a NaN (fmaxf drops it).
__device__ __forceinline__ float amax2(float a, float b) { return (a >= b || a != a) ? a : b; }
__device__ __forceinline__ double amax2(double a, double b) { return (a >= b || a != a) ? a : b; }

// Value of nibble p (bits 4p .. 4p+3) of a word times its scale; exact.
__device__ __forceinline__ float q4_value(uint32_t w, int p, float s) {
  return (float)((int)((w >> (4 * p)) & 15u) - 8) * s;
}

// Weight words: value e (0..7) of a word sits in nibble q4_nibble(e), so that (w >> 4p) & 0x000F000F
// holds the neighbours 2p and 2p + 1 in its two halves.
__host__ __device__ constexpr int q4_nibble(int e) { return (e & 1) ? 4 + e / 2 : e / 2; }

// C[16][8] += A[16][16] B[16][8], bf16 operands, fp32 sums; lane (r, c) = (lane / 4, lane % 4) holds A's rows r
// (a0, a2) and r + 8 (a1, a3), its k pairs 2c (a0, a1) and 2c + 8 (a2, a3), B's column r at the same k pairs (b0,
// b1), and C's rows r (c0, c1) and r + 8 (c2, c3) at columns 2c and 2c + 1.
__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace nsa
