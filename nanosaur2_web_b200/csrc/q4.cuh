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
// Both roundings are decided exactly.  7 s needs eight bits, so 7 s >= amax is an exact comparison, whatever
// amax * (1 / 7) rounded to.  A code is x * inv rounded to an integer, once with inv a little below 1 / s and once a
// little above: where the two agree, so does x / s; where they differ, x / s is next to k + 1/2.  An input of at
// most eight bits (bf16) is then exactly k + 1/2, and the even neighbour is the code; for others the remainder
// x - c s against s / 2 decides, exact because c s needs eight bits and no bit of the remainder, at most about s,
// lies below the lowest of x and c s.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace nsa {

constexpr int kKvGroup = 32;   // values per scale of the cache, along the head dim

template <typename T>
__device__ __forceinline__ float q4_scale(T amax) {
  if (amax < (T)0x1p-110) return 0.f;
  if (!isfinite(amax)) return __uint_as_float(0x7FC00000u);
  const T top = amax < (T)0x1p120 ? amax : (T)0x1p120;
  uint32_t lo = __float_as_uint((float)top * 0.14285715f) & 0xFFF80000u;   // four bits after the leading one
  if ((T)7 * (T)__uint_as_float(lo) < top) lo += 0x00080000u;
  if ((T)7 * (T)__uint_as_float(lo) < top) lo += 0x00080000u;
  return __uint_as_float(lo);
}

// Larger of two magnitudes, a NaN kept.
__device__ __forceinline__ float amax2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ double amax2(double a, double b) { return (a >= b || a != a) ? a : b; }

// Value of nibble p (bits 4p .. 4p+3) of a word times its scale; exact.
__device__ __forceinline__ float q4_value(uint32_t w, int p, float s) {
  return (float)((int)((w >> (4 * p)) & 15u) - 8) * s;
}

// Weight words: value e (0..7) of a word sits in nibble q4_nibble(e), so that (w >> 4p) & 0x000F000F
// holds the neighbours 2p and 2p + 1 in its two halves.
__host__ __device__ constexpr int q4_nibble(int e) { return (e & 1) ? 4 + e / 2 : e / 2; }
// Cache words: value e in nibble e.
__host__ __device__ constexpr int q4_in_order(int e) { return e; }

// Rounding by adding 1.5 * 2^23 (fp64: 1.5 * 2^52) + 8: the low bits of the sum then are c + 8.
__device__ __forceinline__ uint32_t q4_round(float x, float inv) { return __float_as_uint(fmaf(x, inv, 12582920.f)); }
__device__ __forceinline__ uint32_t q4_round(double x, double inv) {
  return (uint32_t)__double2loint(fma(x, inv, 6755399441055752.0));
}

// The slow, exact decision: saturation, and the remainder of x.
template <int N, int (*NIBBLE)(int), typename T>
__device__ __forceinline__ uint32_t q4_bits_exact(const T* x, float s) {
  const T inv = (T)__fdividef(1.f, s), half = (T)0.5 * (T)s;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const T v = x[e] > (T)0x1p120 ? (T)0x1p120 : x[e] < (T)-0x1p120 ? (T)-0x1p120 : x[e];
    uint32_t n = q4_round(v, inv) & 15u;
    const T r = fma((T)(8 - (int)n), (T)s, v);
    if (fabs(r) > half || (fabs(r) == half && (n & 1u))) n += r > (T)0 ? 1u : 0xFFFFFFFFu;
    w += n << (4 * NIBBLE(e));
  }
  return w;
}

// N (4 or 8) stored codes for scale s > 0, value e in nibble NIBBLE(e), from x or, where T is fp64, from its fp32
// roundings xf as far as they decide.  SHORT: every x has at most eight bits.  The nibbles are gathered by adding the
// sums' words times powers of 16; what the sums have above the nibbles adds up to a constant modulo 2^32.
template <int N, int (*NIBBLE)(int), bool SHORT, typename T>
__device__ __forceinline__ uint32_t q4_bits(const T* x, const float* xf, float s, float amax) {
  const float inv = __fdividef(1.f, s), lo = inv * (1.f - 0x1p-20f), hi = inv * (1.f + 0x1p-20f);
  uint32_t w = 0u - 0x4B400000u * (N == 8 ? 0x11111111u : 0x1111u);
  bool slow = !(amax <= 0x1p120f);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const uint32_t a = q4_round(xf[e], lo), b = q4_round(xf[e], hi);
    uint32_t n = a;
    if constexpr (SHORT) {
      n = min(a, b);
      n += n & (a ^ b) & 1u;
    } else {
      slow |= a != b;
    }
    w += n * (1u << (4 * NIBBLE(e)));
  }
  if (slow) w = q4_bits_exact<N, NIBBLE>(x, s);
  return w;
}

// (v & mask) | bits in one instruction (left to the compiler, two constants make it two).
__device__ __forceinline__ uint32_t mask_or(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(v), "r"(mask), "r"(bits));
  return d;
}

// Codes of nibbles P and P + 4 of a word as a bf16 pair, exactly: a nibble n in a bf16 mantissa is 128 + n.
template <int P>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t d;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(mask_or(w >> (4 * P), 0x000F000Fu, 0x43004300u)), "r"(0xC308C308u));
  return d;
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// C[16][8] += A[16][16] B[16][8], bf16 operands, fp32 sums; lane (r, c) = (lane / 4, lane % 4) holds A's rows r
// (a0, a2) and r + 8 (a1, a3), its k pairs 2c (a0, a1) and 2c + 8 (a2, a3), B's column r at the same k pairs (b0,
// b1), and C's rows r (c0, c1) and r + 8 (c2, c3) at columns 2c and 2c + 1.
__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma_bf16_zero(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Asynchronous 16-byte copies to shared memory (shared address, global source).
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {   // all but the N latest groups of this lane are done
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// The first `bytes` (0 or 16) of the source, zeros after them.
__device__ __forceinline__ void copy16_async_fill(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

}  // namespace nsa
