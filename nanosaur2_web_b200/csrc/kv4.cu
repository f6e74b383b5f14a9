// The 4-bit paged key/value cache of a decode step (the format of q4.cuh, groups of 32 along the head
// dim): new tokens normalised, rotated and stored (append), stored tokens read back as bf16 rows, and
// attention over the cache.
//
// Pages: codes [n_pages][2][Hkv][P][D / 2] (keys, then values; value 2j in the low, 2j + 1 in the high
// nibble of byte j), scales [n_pages][2][Hkv][P][D / 32] bf16.  Token t of sequence b is slot t % P of page
// table[b][t / P].  A page id outside the pool, and a position from `cap` on (past the page table, or the RoPE table), is
// recorded in the device error word and its access skipped.
#include <algorithm>

#include <cooperative_groups.h>

#include "nsa_internal.h"
#include "ptx.cuh"
#include "q4.cuh"

namespace nsa {

namespace {

// Page holding position pos (inside the table) of sequence b, or -1 (recorded) when its id is outside the pool.
__device__ __forceinline__ int page_of(const Kv4Params& p, int b, int pos) {
  const int id = p.table[(int64_t)b * p.table_ld + pos / p.P];
  if (id < 0 || id >= p.n_pages) {
    atomicCAS(p.err, 0, kErrKvPage);
    return -1;
  }
  return id;
}

// Index of a token's row: codes at row * D/2 bytes, scales at row * D/32.
__device__ __forceinline__ int64_t cache_row(const Kv4Params& p, int page, int which, int h, int pos) {
  return (((int64_t)page * 2 + which) * p.Hkv + h) * p.P + pos % p.P;
}

// Position of new token i of sequence b; -1 (recorded) when it lies outside.
__device__ __forceinline__ int position(const Kv4Params& p, int b, int i) {
  const int64_t pos = (int64_t)p.start[b] + i;
  if (p.start[b] < 0 || pos >= p.cap) {
    atomicCAS(p.err, 0, kErrKvPosition);
    return -1;
  }
  return (int)pos;
}

// New tokens of sequence b: rows past them are neither read nor written.
__device__ __forceinline__ int new_tokens(const Kv4Params& p, int b) {
  return p.count ? min(max(p.count[b], 0), p.L) : p.L;
}

// Four consecutive inputs.
__device__ __forceinline__ void load4(const float* src, float* x) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(src));
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* src, float* x) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
  x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xFFFF0000u);
  x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xFFFF0000u);
}

// Of one head held by LANES lanes: x[0..3] are elements 4 hl .. of the first half, x[4..7] their partners in the second.
// 1 / rms of the head.
template <typename T, int LANES>
__device__ __forceinline__ T inv_rms(const float* x, float eps) {
  T ss = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += (T)x[e] * (T)x[e];
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if constexpr (sizeof(T) == 8) return rsqrt(ss * (1.0 / (8 * LANES)) + (double)eps);
  else return rsqrtf(ss * (1.f / (8 * LANES)) + eps);
}

// The norm weights with the rotation folded in: out[e] = r (x[e] own[e] + x[e ^ 4] mate[e]).
struct Turn {
  float own[8], mate[8];
};
__device__ __forceinline__ Turn turn_of(const float* w, const float* cs, int64_t sin_off, int64_t row, int half, int hl) {
  Turn t;
  float v[8];
  load4(w + hl * 4, v);
  load4(w + half + hl * 4, v + 4);
  if (cs) {
    float c[4], s[4];
    load4(cs + row * half + hl * 4, c);
    load4(cs + sin_off + row * half + hl * 4, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t.own[e] = v[e] * c[e];
      t.mate[e] = -v[4 + e] * s[e];
      t.own[4 + e] = v[4 + e] * c[e];
      t.mate[4 + e] = v[e] * s[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) t.own[e] = v[e], t.mate[e] = 0.f;
  }
  return t;
}

// A lane's packed codes of its four values of each half and their scales into the head's row of the cache: even lanes
// store the pair's word of the first half, odd lanes that of the second.
__device__ __forceinline__ void store_bits(const uint32_t* bits, const float* s, uint8_t* codes, __nv_bfloat16* scales, int hl,
                                           int half, bool live) {
  const bool odd = hl & 1;
  const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? bits[0] : bits[1], 1);
  if (!live) return;
  const uint32_t word = odd ? got | (bits[1] << 16) : bits[0] | (got << 16);
  *reinterpret_cast<uint32_t*>(codes + (odd ? half / 2 : 0) + hl / 2 * 4) = word;
  if (hl % 8 < 2) scales[(odd ? half / kKvGroup : 0) + hl / 8] = __float2bfloat16_rn(odd ? s[1] : s[0]);
}

// Scales and codes of a lane's values (a group of 32 is eight lanes), from x in T.
template <bool SHORT, typename T>
__device__ __forceinline__ void quantise_halves(const T* x, uint32_t* bits, float* s) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    T am = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) am = amax2((T)fabs(x[4 * k + e]), am);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) am = amax2(__shfl_xor_sync(0xffffffffu, am, o), am);
    s[k] = q4_scale(am);
    if (!(s[k] > 0.f)) bits[k] = 0x8888u;
    else if constexpr (sizeof(T) == 8) bits[k] = q4_bits_exact<4, q4_in_order>(x + 4 * k, s[k]);
    else bits[k] = q4_bits<4, q4_in_order, SHORT>(x + 4 * k, x + 4 * k, s[k], am);
  }
}

// Keys.  The definition is in fp64: the code of a value next to the border of two codes is decided by the last bits, and
// the fp32 order of sums would decide it by chance.  So fp32 decides where its error cannot matter.  The error of a
// value is below 2^-19 r (|x own| + |mate's x mate|): 2^-22 of rsqrtf, half of 15 roundings of the mean square under its
// root, five of the products.  A lane answers false where that is more than 2^-17 of the group's largest magnitude am, where am lies within
// 2^-16 of a border of two scales, or where a code changes within +- 2^-17 am (with 2^-20 of x for 1 / s).  The bound of r
// holds for squares that are normal numbers: with r below 2^50 the mean square is above 2^-101, and what the squares lose
// as subnormals, 2^-150 each, is nothing to it.
__device__ __forceinline__ bool quantise_keys(const float* x, const Turn& t, float r, uint32_t* bits, float* s) {
  bool sure = true;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float v[4], am = 0.f, off = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p0 = x[4 * k + e] * t.own[4 * k + e], p1 = x[4 * (1 - k) + e] * t.mate[4 * k + e];
      v[e] = (p0 + p1) * r;
      off = fmaxf(off, fabsf(p0) + fabsf(p1));
      am = amax2(fabsf(v[e]), am);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) am = amax2(__shfl_xor_sync(0xffffffffu, am, o), am);
    s[k] = q4_scale(am);
    const float below = __uint_as_float(__float_as_uint(s[k]) - 0x00080000u), near = am * 0x1p-16f, step = am * 0x1p-17f;
    sure = sure && off * r * 0x1p-19f <= step && fabsf(7.f * s[k] - am) > near && fabsf(7.f * below - am) > near &&
           am > 0x1p-109f && am < 0x1p119f && r < 0x1p50f;   // (no number: false)
    const float inv = __fdividef(1.f, s[k]), lo = inv * (1.f - 0x1p-20f), hi = inv * (1.f + 0x1p-20f);
    bits[k] = 0u - 0x4B400000u * 0x1111u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t n = q4_round(fabsf(v[e]) - step, lo);   // magnitudes: the code's distance from 8
      sure = sure && n == q4_round(fabsf(v[e]) + step, hi);
      bits[k] += (v[e] < 0.f ? 16u - (n - 0x4B400000u) + 0x4B400000u : n) * (1u << (4 * e));
    }
  }
  return sure;
}

// A CTA per token; a warp takes 256 / D heads of one kind (q, k or v) at a time, eight values a lane.  16 x 500 tokens of
// 32 + 2 x 8 heads of 128: 49.7 us from bf16 (3.5 TB/s), 52.8 us from fp32 (5.1 TB/s).  From bf16 it is half issue and half
// latency: 27 warp instructions per 32 values take 74% of the issue slots, and the longest stall is the wait for a head's
// loads (5.3 of the 13.6 cycles between a warp's instructions).  The launch bound, eight warps in each of six CTAs, holds it
// to 40 registers with 20 to 24 bytes spilled; long calls run four warps a CTA and would not need it.  Loading the next head
// ahead under that bound was slower (72.8 against 64.8 us on an earlier form).
template <typename T, int D>
__global__ void __launch_bounds__(256, 6) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int LANES = D / 8, HPW = 32 / LANES, half = D / 2;
  const Kv4Params& kv = p.kv;
  const int lane = threadIdx.x % 32, hl = lane % LANES, warps = blockDim.x / 32;
  const int q_slots = (p.Hq + HPW - 1) / HPW, kv_slots = (kv.Hkv + HPW - 1) / HPW;
  const int b = blockIdx.x / kv.L, i = blockIdx.x - b * kv.L;
  if (i >= new_tokens(kv, b)) return;
  const int pos = position(kv, b, i);
  if (pos < 0) return;
  const T* row = static_cast<const T*>(p.qkv) + b * p.bstride + i * p.ld + hl * 4;
  int slot = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  if (slot < q_slots) {
    const Turn t = turn_of(p.q_w, p.cs, p.sin_off, pos, half, hl);
    __nv_bfloat16* out = p.q_out + b * p.qo_bstride + i * p.qo_ld + hl * 4;
    for (; slot < q_slots; slot += warps) {
      const int h = slot * HPW + lane / LANES;
      const bool live = h < p.Hq;                                  // lanes past the last head repeat it, storing nothing
      const int at = (live ? h : p.Hq - 1) * D;
      float x[8], o[8];
      load4(row + p.q_off + at, x);
      load4(row + p.q_off + at + half, x + 4);
      float r = inv_rms<float, LANES>(x, p.eps);
      // squares that are infinite, or so small that subnormal ones weigh, are taken of the head times a power of two
      if (__any_sync(0xffffffffu, !(r > 0.f && r < 0x1p50f))) {
        const float c = r >= 0x1p50f ? 0x1p100f : r > 0.f ? 1.f : 0x1p-70f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= c;
        r = inv_rms<float, LANES>(x, p.eps * c * c);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmaf(x[e ^ 4], t.mate[e], x[e] * t.own[e]) * r;
      if (live) {
        *reinterpret_cast<uint2*>(out + at) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
        *reinterpret_cast<uint2*>(out + at + half) = make_uint2(pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
      }
    }
  }
  if (slot >= q_slots + 2 * kv_slots) return;
  const int page = page_of(kv, b, pos);
  if (page < 0) return;
  for (slot -= q_slots; slot < 2 * kv_slots; slot += warps) {
    const int which = slot < kv_slots ? 0 : 1;
    const int h = (slot - which * kv_slots) * HPW + lane / LANES;
    const bool live = h < kv.Hkv;
    const int hh = live ? h : kv.Hkv - 1;
    const int64_t tok = cache_row(kv, page, which, hh, pos);
    uint8_t* codes = kv.codes + tok * (D / 2);
    __nv_bfloat16* scales = kv.scales + tok * (D / kKvGroup);
    const T* src = row + (which ? p.v_off : p.k_off) + (int64_t)hh * D;
    float x[8], s[2];
    uint32_t bits[2];
    load4(src, x);
    load4(src + half, x + 4);
    if (which) {
      quantise_halves<sizeof(T) == 2>(x, bits, s);
    } else {
      const Turn t = turn_of(p.k_w, p.cs, p.sin_off, pos, half, hl);
      if (__any_sync(0xffffffffu, !quantise_keys(x, t, inv_rms<float, LANES>(x, p.eps), bits, s))) {
        float w[8], c[4], sn[4];
        double y[8];
        load4(p.k_w + hl * 4, w);
        load4(p.k_w + half + hl * 4, w + 4);
        const double r = inv_rms<double, LANES>(x, p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (double)x[e] * r * (double)w[e];
        if (p.cs) {
          load4(p.cs + (int64_t)pos * half + hl * 4, c);
          load4(p.cs + p.sin_off + (int64_t)pos * half + hl * 4, sn);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double a = y[e], b2 = y[4 + e];
            y[e] = a * (double)c[e] - b2 * (double)sn[e];
            y[4 + e] = b2 * (double)c[e] + a * (double)sn[e];
          }
        }
        quantise_halves<false>(y, bits, s);
      }
    }
    store_bits(bits, s, codes, scales, hl, half, live);
  }
}

// A CTA per R rows, a thread per word (8 values) of each: the rows' loads are under way together.  16 x 500 tokens of 8 heads
// of 128 take 15.3 us (2.7 TB/s): a chain of start, table, codes and stores for little work per thread (72% of the issue
// slots, 4.0 of 18.5 cycles per instruction waiting for loads).
template <int R>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Params p, __nv_bfloat16* __restrict__ out, int64_t ldo,
                                                       int64_t bstride) {
  const int words = p.D / 8, shift = 31 - __clz(words);
  int64_t tok[R], to[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int64_t row = (int64_t)blockIdx.x * R + k;
    tok[k] = -1;
    if (row >= (int64_t)p.B * p.L) continue;
    const int b = (int)(row / p.L), i = (int)(row - (int64_t)b * p.L);
    if (i >= new_tokens(p, b)) continue;
    const int pos = position(p, b, i);
    if (pos < 0) continue;
    const int page = page_of(p, b, pos);
    if (page < 0) continue;
    tok[k] = cache_row(p, page, 0, 0, pos);
    to[k] = b * bstride + i * ldo;
  }
  for (int e = threadIdx.x; e < 2 * p.Hkv * words; e += blockDim.x) {
    const int w = e & (words - 1), h = e >> shift;                 // h: key heads, then value heads, P rows apart
    uint32_t v[R], s2[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (tok[k] < 0) continue;
      const int64_t at = tok[k] + (int64_t)h * p.P;
      v[k] = __ldg(reinterpret_cast<const uint32_t*>(p.codes + at * (p.D / 2)) + w);
      s2[k] = __ldg(reinterpret_cast<const uint16_t*>(p.scales) + at * (p.D / kKvGroup) + w / 4) * 0x10001u;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (tok[k] < 0) continue;
      const uint32_t v04 = mul_bf16x2(code_pair<0>(v[k]), s2[k]), v15 = mul_bf16x2(code_pair<1>(v[k]), s2[k]);
      const uint32_t v26 = mul_bf16x2(code_pair<2>(v[k]), s2[k]), v37 = mul_bf16x2(code_pair<3>(v[k]), s2[k]);
      uint4 o;
      o.x = __byte_perm(v04, v15, 0x5410);
      o.y = __byte_perm(v26, v37, 0x5410);
      o.z = __byte_perm(v04, v15, 0x7632);
      o.w = __byte_perm(v26, v37, 0x7632);
      reinterpret_cast<uint4*>(out + to[k])[e] = o;
    }
  }
}

// ------------------------------------------------------------------------------------ attention
//
// A unit is 8 or 16 query rows that share a key/value head (row R of sequence b is new token R / group, query head
// R % group of the head's group) over the blocks of 16 tokens that they see (a block never straddles pages).  The
// blocks of all units in a row are dealt out evenly to one wave of CTAs, whatever the sequences' lengths, so a CTA works
// on the end of one unit, some whole ones and the beginning of another.  Within a CTA each warp walks its own blocks
// with its own running maximum, sum and output, joined in shared memory; what CTAs have of a shared unit is joined
// by a second kernel.  Few and short units are latency instead: a cluster of eight CTAs takes one unit and joins it
// through its shared memories.  The host chooses, and by what it knows: the page table's width, not the sequences' lengths.
//
// Both products run on mma.m16n8k16 with the cached operand as A, so that the eight query rows fill N = 8 and
// only the cache's bytes are converted:
//   S^T [16 tokens][8 rows] = K [16 tokens][D] Q^T,   O^T [D][8 rows] += V^T [D][16 tokens] P^T.
// A tcgen05 tile would need the converted operand in shared memory (4 times the cache's bytes written and
// read again there); here the blocks themselves are brought there, a few ahead of their use, and each lane reads its
// 4-bit words in the A fragment's own order, converts them in registers and multiplies.  The contraction index of a product may be permuted, so
// lane (r, c) = (lane / 4, lane % 4) takes, of token r, the 16-byte pieces c of the row: nibbles p and p + 4
// of a word are one bf16 pair, and Q is staged in the matching order.  For V the lane takes piece r of the
// tokens 2c, 2c + 1, 2c + 8, 2c + 9 (what its B fragment of P^T holds) and pairs the tokens' words by byte
// permutes; the rows of an output tile are the lane's own dims.  Conversion: a nibble n moved to the top of a
// bf16 mantissa is 1 + n / 16, and (1 + n / 16) 16 s - 24 s = s (n - 8) is one bf16x2 fma, exact because the
// scale has five significant bits (q4.cuh).
//
// P^T is P's accumulator transposed: packed to bf16 and turned by movmatrix.  P is split into two bf16 terms
// (16 bits together): one bf16 would add an error as large as the output's own rounding.  Where a unit has at most four
// rows, half of the columns would be empty: they take the same rows again, the scores there are the same, and the low
// terms are what they multiply the values with, so that one product does for both.
//
// What bounds it is the issue of instructions: an mma.m16n8k16 holds a scheduler for about 5 cycles (and its tensor unit
// for 8), a pair of converted values costs 3 instructions, two of them at half rate.  On a form that took 71.9 us for 8192
// blocks of 8 heads and 16 rows (D 128; 63.5 us now), 71.2 without the copies and 39.8 without the products and
// conversions.  Two blocks at a time give the scheduler independent chains (D 256: 33.2 -> 29.7 us at 8 x 32768 tokens)
// and share the walk, the tests of masks and maxima (466 instead of 594 instructions a block).
// The running maximum moves only when a score exceeds it by 2^8 in the exponent's base, which spares a reduction over
// lanes per block.  What is subtracted from the scores is the maximum and `shift` more, ceil(log2(tokens a row may see))
// + 1, so that the weights of a row sum to at most 2^7 and the unnormalised outputs of the largest values, 2^120, stay finite.

constexpr int kAttnWarps = 4;       // with 8, a call over 1024 tokens took 10.6 us instead of 7.7
constexpr int kAtOnce = 2;          // blocks that a warp takes at a time
constexpr int kSetup = 20;          // what another unit costs a CTA, in blocks (0, 8, 20, 32: 69.6, 67.6, 64.3, 64.9 us
                                    // at 4 tokens over 131071; 74.7, 73.0, 72.5, 72.6 us at 40 sequences up to 8192)
constexpr float kMaxSlack = 8.f;   // exp2 of a score may reach 2^8 before the maximum is moved

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// 16 s and -24 s of a pair of scales.
struct ScalePair {
  uint32_t s16, m24;
};
__device__ __forceinline__ ScalePair scale_pair(uint32_t lo, uint32_t hi) {
  const uint32_t s = lo | (hi << 16);
  return {mul_bf16x2(s, 0x41804180u), mul_bf16x2(s, 0xC1C0C1C0u)};
}

// Nibble P of both halves of x times its scale.
template <int P>
__device__ __forceinline__ uint32_t dequant(uint32_t x, ScalePair s) {
  const uint32_t m = P == 0 ? x << 3 : x >> (4 * P - 3);
  return fma_bf16x2(mask_or(m, 0x00780078u, 0x3F803F80u), s.s16, s.m24);
}

// N 32-bit words (1, 2 or 4 aligned), or a scale, from shared memory.
template <int N>
__device__ __forceinline__ void load_words(uint32_t at, uint32_t* w) {
  if constexpr (N == 1)
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
  else
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
}
__device__ __forceinline__ uint32_t load_scale(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}

// Which 16-token blocks the rows at positions pmin .. pmax see: [0, sink_blocks), then from first on; n in all.
struct Blocks {
  int sink_blocks, first, n;
};
__device__ __forceinline__ Blocks blocks_of(int pmin, int pmax, int window, int sinks) {
  const int lo = window > 0 ? max(0, pmin - window + 1) : 0;
  const int first = lo / 16;
  const int ns = min((min(sinks, lo) + 15) / 16, first);
  return {ns, first, ns + pmax / 16 - first + 1};
}

// New token of row R of a sequence's rows.
__device__ __forceinline__ int token_of(const Kv4Params& kv, int R, int group) { return kv.L == 1 ? 0 : R / group; }

// The rows of row tile rt of sequence b: new tokens i_first .. i_last (none: i_last < i_first) at positions pmin .. pmax;
// outside: some of them lie outside and see nothing.
struct Tile {
  int row0, rows, i_first, i_last, pmin, pmax;
  bool outside;
  Blocks bl;
};
__device__ __forceinline__ Tile tile_of(const Kv4AttnParams& p, int b, int rt, int rows_per_tile, int group) {
  const Kv4Params& kv = p.kv;
  Tile t;
  t.row0 = rt * rows_per_tile;
  t.rows = min(rows_per_tile, kv.L * group - t.row0);
  t.i_first = token_of(kv, t.row0, group);
  t.i_last = min(token_of(kv, t.row0 + t.rows - 1, group), new_tokens(kv, b) - 1);
  const int64_t start = kv.start[b], cap = kv.cap;
  t.outside = t.i_last >= t.i_first && (start < 0 || start + t.i_last >= cap);
  t.pmin = (int)(start + t.i_first);
  t.pmax = (int)min(start + t.i_last, cap - 1);
  t.bl = {0, 0, 0};
  if (t.i_last >= t.i_first && start >= 0 && start + t.i_first < cap && kv.n_pages > 0)
    t.bl = blocks_of(t.pmin, t.pmax, p.window, p.sinks);
  return t;
}
// Blocks of a unit of the tile; a unit that sees nothing but has rows to write counts one.
__device__ __forceinline__ int unit_blocks(const Tile& t) { return t.i_last < t.i_first ? 0 : max(t.bl.n, 1); }

// A block of 16 tokens in shared memory: keys, values (8 D bytes each), key scales, value scales (D bytes each).  The
// 16-byte pieces of the codes are moved within each 128 bytes so that neither the keys' reads (all pieces of eight
// tokens) nor the values' (one piece of every other token) meet on a bank.
template <int D>
struct Stage {
  static constexpr int values = 8 * D, scales = 16 * D, bytes = 18 * D;
  static constexpr int copies = D / 64;   // pieces of the keys (and of the values) per lane
  // place of piece q of token t
  static __device__ __forceinline__ int at(int t, int q) {
    constexpr int per = D / 32;           // pieces per token
    const int e = t * per + q, row = e / 8, x = e % 8;
    const int f = D == 256 ? ((row >> 1) & 3) * 2 ^ (row & 1) * 4 : D == 128 ? (row & 3) * 2 : (row & 1) * 2;
    return row * 128 + (x ^ f) * 16;
  }
};

template <int D, int NT>
struct AttnSmem {
  static constexpr int stages = D == 256 ? 4 : 6;
  static constexpr size_t q = (size_t)D / 16 * NT * 32 * 8;                         // Q^T fragments
  static constexpr size_t ring = (size_t)kAttnWarps * stages * Stage<D>::bytes;
  static constexpr size_t o = (size_t)kAttnWarps * 8 * NT * (D + 4) * 4;            // warps' outputs, rows padded
  static constexpr size_t ml = (size_t)kAttnWarps * 8 * NT * 2 * 4;                 // ... and their (m, l)
  static constexpr size_t bytes = (q + ring > o ? q + ring : o) + ml;
};

// As many as registers and shared memory hold.  More (4 and 5 of fewer registers) took 80.7 and 84.8 us where 3 took 78.7.
constexpr int ctas_per_sm(int D, int NT) { return NT == 1 && D < 256 ? 3 : 2; }

// NT: tiles of eight query rows; SPLIT: one tile of at most four, whose columns 4 .. 7 are its rows again.  CL: 1, or the
// CTAs of a cluster that takes one unit.
template <int D, int NT, bool SPLIT, int CL>
__global__ void __launch_bounds__(kAttnWarps * 32, ctas_per_sm(D, NT)) kv4_attention_kernel(const Kv4AttnParams p) {
  constexpr int KW = D / 32;   // words of a token's keys per lane
  constexpr int VW = D / 64;   // words of a token's values per lane
  constexpr int KG = D == 256 ? 2 : 1;
  constexpr int ROWS = 8 * NT, STAGES = AttnSmem<D, NT>::stages, U = kAtOnce;
  extern __shared__ __align__(16) uint8_t smem[];
  const Kv4Params& kv = p.kv;
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);   // known to be the same in all lanes
  const int group = p.Hq / kv.Hkv;

  // this CTA's blocks [g0, g1) of all units' (units: sequence, row tile, kv head), and the (sequence, tile) of the first
  int g0 = 0, g1 = 1, per = 1, entry = 0, before = 0;   // before: blocks of the entries before
  if constexpr (CL == 1) {
    const int tiles = kv.B * p.row_tiles;
    const auto blocks_at = [&](int e) {
      const int n = e < tiles ? unit_blocks(tile_of(p, e / p.row_tiles, e % p.row_tiles, ROWS, group)) : 0;
      return n ? kv.Hkv * (n + kSetup) : 0;
    };
    int own = blocks_at(lane), total = __reduce_add_sync(0xffffffffu, own);
    for (int e0 = 32; e0 < tiles; e0 += 32) total += __reduce_add_sync(0xffffffffu, blocks_at(e0 + lane));
    per = max((total - 1) / (int)gridDim.x + 1, kAttnWarps);
    g0 = (int)min((int64_t)blockIdx.x * per, (int64_t)total);
    g1 = min(g0 + per, total);
    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) p.part_head[blockIdx.x] = make_int2(-1, 0);
    if (g0 >= g1) return;
    for (int e0 = 0;; e0 += 32) {
      if (e0 > 0) own = blocks_at(e0 + lane);
      int upto = own;
  #pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > g0);
      if (hit) {
        const int src = __ffs(hit) - 1;
        entry = e0 + src;
        before += __shfl_sync(0xffffffffu, upto - own, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  } else {
    entry = blockIdx.x / CL / kv.Hkv;
  }

  // Where blocks are: 16 tokens of a head are 8 D bytes of codes and D of scales, so a 32-bit index of blocks and one
  // wide multiply-add give every address.  A lane copies pieces lane, lane + 32, .. of the codes; of the scales, the
  // first D / 16 lanes the keys' and the next D / 16 the values'.
  const uint32_t ppb = kv.P / 16, to_values = kv.Hkv * ppb;
  const uint8_t* codes = kv.codes + lane * 16;
  const bool copies_scales = lane < D / 8, value_scales = lane >= D / 16;
  const uint8_t* scales = reinterpret_cast<const uint8_t*>(kv.scales) + (value_scales ? (uint64_t)to_values * D : 0) + lane % (D / 16) * 16;
  const uint32_t ring_at = smem_u32(smem + AttnSmem<D, NT>::q) + warp * STAGES * Stage<D>::bytes;
  uint32_t code_at[Stage<D>::copies];
#pragma unroll
  for (int x = 0; x < Stage<D>::copies; ++x) {
    const int e = lane + 32 * x;
    code_at[x] = Stage<D>::at(e / (D / 32), e % (D / 32));
  }
  const uint32_t scale_at = Stage<D>::scales + (value_scales ? D : 0) + lane % (D / 16) * 16;
  // what the lane reads of a stage: its key words of tokens r and r + 8, value words of tokens 2c, 2c + 1, 2c + 8, 2c + 9
  // (eight tokens on is 4 D bytes on, pieces moved alike)
  uint32_t k_at[KW > 4 ? 2 : 1], v_at[2];
#pragma unroll
  for (int y = 0; y < (KW > 4 ? 2 : 1); ++y) k_at[y] = D == 64 ? Stage<D>::at(r, c / 2) + c % 2 * 8 : Stage<D>::at(r, c + 4 * y);
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int t = 2 * c + x;
    v_at[x] = Stage<D>::values + (D == 256 ? Stage<D>::at(t, r) : D == 128 ? Stage<D>::at(t, r / 2) + r % 2 * 8 : Stage<D>::at(t, r / 4) + r % 4 * 4);
  }
  const uint32_t ks_at = Stage<D>::scales + r * (D / 16) + 2 * (D == 64 ? c / 2 : c);
  const uint32_t vs_at = Stage<D>::scales + D + 2 * c * (D / 16) + r * VW / 4 * 2;

  for (int g = g0; g < g1;) {
  const int b = entry / p.row_tiles, rt = entry % p.row_tiles;
  const Tile tl = tile_of(p, b, rt, ROWS, group);
  const Blocks bl = tl.bl;
  const int n = unit_blocks(tl);
  int hk, first, last, begins = 0;   // this CTA's blocks of the unit: [first, last); where the unit begins
  if constexpr (CL == 1) {
    const int all = n ? n + kSetup : 0;
    if (g - before >= kv.Hkv * all) {   // on to the next tile with rows
      before += kv.Hkv * all;
      ++entry;
      continue;
    }
    hk = (g - before) / all;
    begins = before + hk * all;
    first = max(g - begins - kSetup, 0);
    last = min(n, g1 - begins - kSetup);
    if (last <= 0) return;   // no more than the unit's set-up: the next CTA has its first block
  } else {
    if (n == 0) return;   // the whole cluster
    hk = blockIdx.x / CL % kv.Hkv;
    const int share = (n + CL - 1) / CL;
    first = min((int)(blockIdx.x % CL) * share, n);
    last = min(first + share, n);
  }
  const int row0 = tl.row0, rows = tl.rows, i_last = tl.i_last, pmin = tl.pmin, pmax = tl.pmax;
  if (threadIdx.x == 0 && first == 0 && last > 0 && hk == 0) {
    if (tl.outside) atomicCAS(kv.err, 0, kErrKvPosition);
    else if (kv.n_pages == 0) atomicCAS(kv.err, 0, kErrKvPage);
  }
  // this warp's blocks
  const int each = (last - first + kAttnWarps - 1) / kAttnWarps;
  const int ta = min(first + warp * each, last), tb = bl.n > 0 ? min(ta + each, last) : ta;
  const int* table = kv.table + (int64_t)b * kv.table_ld;

  // The rows of Q, 16 bytes (a word's dims) a thread at a time; under way while the first blocks are.
  constexpr int Q = (KW * NT + kAttnWarps - 1) / kAttnWarps;
  uint4 qv[Q];
#pragma unroll
  for (int x = 0; x < Q; ++x) {
    const int e = threadIdx.x + x * kAttnWarps * 32, ln = e % 32, cc = ln % 4, w = e / 32 / NT;
    const int rr = SPLIT ? ln / 4 % 4 : 8 * (e / 32 % NT) + ln / 4;
    const int word = D == 256 ? 4 * (cc + 4 * (w / 4)) + w % 4 : KW * cc + w;
    const int i = token_of(kv, row0 + rr, group);
    qv[x] = make_uint4(0u, 0u, 0u, 0u);
    if (e < KW * NT * 32 && rr < rows && i <= i_last)
      qv[x] = __ldg(reinterpret_cast<const uint4*>(p.q + b * p.q_bstride + i * p.q_ld + (int64_t)(hk * group + row0 + rr - i * group) * D + word * 8));
  }

  // Walks the warp's blocks, STAGES - U ahead of their use: `at` and `left` are the next block's index and the blocks
  // until another page (or the jump from the first tokens to the window).  A missing page stands on page 0, masked
  // (`absent`, one bit per stage).  The ids of the two pages ahead are loaded early.
  int w_t, left, id1, id2;
  uint32_t at, w_page, absent;
  bool missing;
  const auto id_of = [&](uint32_t page) { return page < (uint32_t)kv.max_pages ? __ldg(table + page) : -1; };
  const auto enter = [&](int id, uint32_t slot) {   // page w_page from its block `slot` on
    missing = id < 0 || id >= kv.n_pages;
    if (missing && lane == 0) atomicCAS(kv.err, 0, kErrKvPage);
    at = ((uint32_t)(missing ? 0 : id) * 2 * kv.Hkv + hk) * ppb + slot;
    left = (int)(ppb - slot);
    if (w_t < bl.sink_blocks) left = min(left, bl.sink_blocks - w_t);
  };
  const auto jump = [&] {   // to block w_t, wherever it is
    const uint32_t blk = w_t < bl.sink_blocks ? w_t : bl.first + w_t - bl.sink_blocks;
    w_page = blk / ppb;
    const int id = id_of(w_page);
    id1 = id_of(w_page + 1);
    id2 = id_of(w_page + 2);
    enter(id, blk - w_page * ppb);
  };
  const auto fetch = [&](int st) {   // block w_t into stage st, then on to the next
    if (w_t < tb) {
      if (left == 0) {
        if (w_t == ta || w_t == bl.sink_blocks) {
          jump();
        } else {
          ++w_page;
          const int id = id1;
          id1 = id2;
          id2 = id_of(w_page + 2);
          enter(id, 0);
        }
      }
      const uint32_t to = ring_at + st * Stage<D>::bytes;
      const uint8_t* k = codes + (uint64_t)at * (8 * D);
      const uint8_t* v = codes + (uint64_t)(at + to_values) * (8 * D);
#pragma unroll
      for (int x = 0; x < Stage<D>::copies; ++x) copy16_async(to + code_at[x], k + 512 * x);
      if (copies_scales) copy16_async(to + scale_at, scales + (uint64_t)at * D);
#pragma unroll
      for (int x = 0; x < Stage<D>::copies; ++x) copy16_async(to + Stage<D>::values + code_at[x], v + 512 * x);
      if (missing || absent) absent = (absent & ~(1u << st)) | ((uint32_t)missing << st);
      ++w_t;
      ++at;
      --left;
    }
    copy_commit();
  };
  const auto begin = [&] {
    w_t = ta;
    left = 0;
    absent = 0;
#pragma unroll
    for (int st = 0; st < STAGES - U; ++st) fetch(st);
  };
  begin();

  int pos[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = SPLIT ? (2 * c + j) % 4 : 8 * t + 2 * c + j, i = token_of(kv, row0 + k, group);
      pos[t][j] = k < rows && i <= i_last && bl.n > 0 && pmin + (i - tl.i_first) <= pmax ? pmin + (i - tl.i_first) : -1;
    }
  // every row sees every token of the blocks numbered [whole0, whole1)
  const int whole0 = p.window > 0 ? bl.sink_blocks + (max(pmax - p.window + 1, 0) + 15) / 16 - bl.first : 0;
  const int jump_by = 16 * (bl.first - bl.sink_blocks);
  const int whole1 = tl.outside ? 0 : bl.sink_blocks + (pmin + 1) / 16 - bl.first;

  // Q^T fragments: for k-step 2w + s of lane (r, c), words of row r's dims in the order of the lane's key words
  uint2* qs = reinterpret_cast<uint2*>(smem);
#pragma unroll
  for (int x = 0; x < Q; ++x) {
    const int e = threadIdx.x + x * kAttnWarps * 32, ln = e % 32, t = e / 32 % NT, w = e / 32 / NT;
    if (e >= KW * NT * 32) break;
    // pairs (e, e + 4): e = 2 s and 2 s + 1
    qs[(2 * w * NT + t) * 32 + ln] = make_uint2(__byte_perm(qv[x].x, qv[x].z, 0x5410), __byte_perm(qv[x].x, qv[x].z, 0x7632));
    qs[((2 * w + 1) * NT + t) * 32 + ln] = make_uint2(__byte_perm(qv[x].y, qv[x].w, 0x5410), __byte_perm(qv[x].y, qv[x].w, 0x7632));
  }
  __syncthreads();

  // m: the largest raw score so far; lim: what a score may reach before m moves; z: the scaled maximum + shift, which is
  // subtracted (0 while there is none)
  const float slack = kMaxSlack / p.scale_log2;
  float o[NT][VW * 4][4], m[NT][2], lim[NT][2], z[NT][2], l[NT][2];
  // The second pass, only after an output that is not a number: see `careful` below.
  for (bool careful = false;; careful = true) {
    if (careful) begin();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int x = 0; x < VW * 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[t][x][y] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) m[t][j] = lim[t][j] = -INFINITY, z[t][j] = 0.f, l[t][j] = 0.f;
    }
    int stage = 0;
    for (int tt = ta; tt < tb; tt += U) {
      copy_wait<STAGES - 2 * U>();
      __syncwarp();   // the blocks are there for all lanes, and all lanes are done with the stages that are filled next
#pragma unroll
      for (int u = 0; u < U; ++u) fetch((stage == 0 ? STAGES - U : stage - U) + u);
      const uint32_t blk = ring_at + stage * Stage<D>::bytes;
      // first token of each block; past the warp's last block, and where a page is missing, there is nothing
      int j_now[U];
      bool gone[U], part = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        j_now[u] = 16 * (tt + u) + (tt + u < bl.sink_blocks ? 0 : jump_by);
        gone[u] = (absent && (absent >> (stage + u) & 1)) || tt + u >= tb;
        part = part || tt + u < whole0 || tt + u >= whole1 || gone[u];
      }
      stage = stage == STAGES - U ? 0 : stage + U;
      float x[U][NT][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t kw[2][KW], ks[2][KG];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t at = blk + u * Stage<D>::bytes;
          load_words<(KW > 4 ? 4 : KW)>(at + k_at[0] + h * 4 * D, kw[h]);
          if constexpr (KW > 4) load_words<4>(at + k_at[1] + h * 4 * D, kw[h] + 4);
#pragma unroll
          for (int y = 0; y < KG; ++y) ks[h][y] = load_scale(at + ks_at + h * (D / 2) + 8 * y);
        }
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const int g2 = KG == 2 ? w / 4 : 0;
          const ScalePair sa = scale_pair(ks[0][g2], ks[0][g2]), sb = scale_pair(ks[1][g2], ks[1][g2]);
          const uint32_t a0 = dequant<0>(kw[0][w], sa), a1 = dequant<0>(kw[1][w], sb), a2 = dequant<1>(kw[0][w], sa),
                         a3 = dequant<1>(kw[1][w], sb), a4 = dequant<2>(kw[0][w], sa), a5 = dequant<2>(kw[1][w], sb),
                         a6 = dequant<3>(kw[0][w], sa), a7 = dequant<3>(kw[1][w], sb);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint2 q0 = qs[(2 * w * NT + t) * 32 + lane], q1 = qs[((2 * w + 1) * NT + t) * 32 + lane];
            if (w == 0) mma_bf16_zero(x[u][t], a0, a1, a2, a3, q0.x, q0.y);
            else mma_bf16(x[u][t], a0, a1, a2, a3, q0.x, q0.y);
            mma_bf16(x[u][t], a4, a5, a6, a7, q1.x, q1.y);
          }
        }
      }
      uint32_t vw[U][4][VW], vs[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t at = blk + u * Stage<D>::bytes;
          load_words<VW>(at + v_at[y & 1] + (y >> 1) * 4 * D, vw[u][y]);
          vs[u][y] = load_scale(at + vs_at + ((y & 1) + 8 * (y >> 1)) * (D / 16));
        }
      const auto see = [&](int u, int ps, int j) {
        return !gone[u] && j <= ps && (p.window == 0 || j > ps - p.window || j < p.sinks);
      };
      if (__any_sync(0xffffffffu, part)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (!see(u, pos[t][y & 1], j_now[u] + r + 8 * (y >> 1))) x[u][t][y] = -INFINITY;
          // tokens no row sees may hold anything: their values become zeros
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int j = j_now[u] + 2 * c + (y & 1) + 8 * (y >> 1);
            if (gone[u] || j > pmax || (p.window > 0 && j <= pmin - p.window && j >= p.sinks)) vs[u][y] = 0;
          }
        }
      }
      float top[NT][2];
      bool up = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[t][j] = fmaxf(fmaxf(x[0][t][j], x[0][t][j + 2]), fmaxf(x[1][t][j], x[1][t][j + 2]));
          up |= top[t][j] > lim[t][j];
        }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float f[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float n2 = top[t][j];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) n2 = fmaxf(n2, __shfl_xor_sync(0xffffffffu, n2, d));
            n2 = fmaxf(n2, m[t][j]);
            const float old = z[t][j];
            z[t][j] = n2 == -INFINITY ? 0.f : fmaf(n2, p.scale_log2, p.shift);
            f[j] = m[t][j] == -INFINITY ? 0.f : ex2(old - z[t][j]);
            m[t][j] = n2;
            lim[t][j] = n2 == -INFINITY ? n2 : n2 + slack;
            l[t][j] *= f[j];
          }
#pragma unroll
          for (int y = 0; y < VW * 4; ++y) {
            o[t][y][0] *= f[0]; o[t][y][1] *= f[1];
            o[t][y][2] *= f[0]; o[t][y][3] *= f[1];
          }
        }
      }
      uint32_t ph[U][NT][2], pl[U][NT][2];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float* e = x[u][t];
#pragma unroll
          for (int y = 0; y < 4; ++y) e[y] = ex2(fmaf(e[y], p.scale_log2, -z[t][y & 1]));
          l[t][0] += e[0] + e[2];
          l[t][1] += e[1] + e[3];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t hi = pack_bf16x2(e[2 * y], e[2 * y + 1]);
            const uint32_t lo = pack_bf16x2(e[2 * y] - __uint_as_float(hi << 16), e[2 * y + 1] - __uint_as_float(hi & 0xFFFF0000u));
            ph[u][t][y] = transpose8x8(SPLIT && c >= 2 ? lo : hi);
            if constexpr (!SPLIT) pl[u][t][y] = transpose8x8(lo);
          }
        }
      // A value group with an infinity or a NaN is NaN in the outputs of the rows that see it; as a factor it
      // reaches the others of the tile too (0 * NaN).  Where an output came out as no number the blocks are walked
      // again with such groups taken out of the product and added to their rows here.
      if (careful) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          for (int k = 0; k < 16; ++k) {
            const int y = (k & 1) + 2 * (k >> 3), src = r * 4 + (k % 8) / 2;
            const uint32_t own = y == 0 ? vs[u][0] : y == 1 ? vs[u][1] : y == 2 ? vs[u][2] : vs[u][3];
            const uint32_t sk = __shfl_sync(0xffffffffu, own, src);
            if ((sk & 0x7F80u) != 0x7F80u) continue;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (see(u, pos[t][j], j_now[u] + k)) {
#pragma unroll
                  for (int w = 0; w < VW * 4; ++w) o[t][w][j] = o[t][w][j + 2] = __uint_as_float(0x7FC00000u);
                }
          }
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if ((vs[u][y] & 0x7F80u) == 0x7F80u) vs[u][y] = 0;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const ScalePair va = scale_pair(vs[u][0], vs[u][1]), vb = scale_pair(vs[u][2], vs[u][3]);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t xa = __byte_perm(vw[u][0][w], vw[u][1][w], 0x5410), ya = __byte_perm(vw[u][0][w], vw[u][1][w], 0x7632);
          const uint32_t xb = __byte_perm(vw[u][2][w], vw[u][3][w], 0x5410), yb = __byte_perm(vw[u][2][w], vw[u][3][w], 0x7632);
          const auto tile = [&](int x4, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma_bf16(o[t][x4], a0, a1, a2, a3, ph[u][t][0], ph[u][t][1]);
              if constexpr (!SPLIT) mma_bf16(o[t][x4], a0, a1, a2, a3, pl[u][t][0], pl[u][t][1]);
            }
          };
          tile(4 * w + 0, dequant<0>(xa, va), dequant<0>(ya, va), dequant<0>(xb, vb), dequant<0>(yb, vb));
          tile(4 * w + 1, dequant<1>(xa, va), dequant<1>(ya, va), dequant<1>(xb, vb), dequant<1>(yb, vb));
          tile(4 * w + 2, dequant<2>(xa, va), dequant<2>(ya, va), dequant<2>(xb, vb), dequant<2>(yb, vb));
          tile(4 * w + 3, dequant<3>(xa, va), dequant<3>(ya, va), dequant<3>(xb, vb), dequant<3>(yb, vb));
        }
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int y = 0; y < VW * 4; ++y) sum += (o[t][y][0] - o[t][y][0]) + (o[t][y][1] - o[t][y][1]) + (o[t][y][2] - o[t][y][2]) + (o[t][y][3] - o[t][y][3]);
    if (careful || !__any_sync(0xffffffffu, sum != 0.f)) break;   // x - x is 0 unless x is infinite or no number
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], d);

  // join the warps
  copy_wait<0>();
  __syncthreads();   // nothing reads the fragments of Q or the ring any more
  float* so = reinterpret_cast<float*>(smem);
  float* sm = reinterpret_cast<float*>(smem + AttnSmem<D, NT>::bytes - AttnSmem<D, NT>::ml);
  constexpr int LD = D + 4;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int k = warp * ROWS + 8 * t + 2 * c;
    if constexpr (SPLIT) {   // columns 4 .. 7 have what P's low parts gave
#pragma unroll
      for (int x = 0; x < VW * 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[t][x][y] += __shfl_down_sync(0xffffffffu, o[t][x][y], 2);
      if (c >= 2) continue;
    }
#pragma unroll
    for (int w = 0; w < VW; ++w)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float* d = so + k * LD + 8 * (VW * r + w) + x;
        d[0] = o[t][4 * w + x][0];
        d[LD] = o[t][4 * w + x][1];
        d[4] = o[t][4 * w + x][2];
        d[LD + 4] = o[t][4 * w + x][3];
      }
    if (r == 0) {
      float* ml = sm + k * 2;
      ml[0] = m[t][0] == -INFINITY ? m[t][0] : z[t][0]; ml[1] = l[t][0];
      ml[2] = m[t][1] == -INFINITY ? m[t][1] : z[t][1]; ml[3] = l[t][1];
    }
  }
  // every warp of the CTA, or of the cluster's CTAs
  namespace cg = cooperative_groups;
  if constexpr (CL > 1) cg::this_cluster().sync();
  else __syncthreads();
  const int from = CL > 1 ? (blockIdx.x % CL) * kAttnWarps * 32 + threadIdx.x : threadIdx.x;
  for (int e = from; e < rows * (D / 4); e += CL * kAttnWarps * 32) {
    const int k = e / (D / 4), d = e % (D / 4) * 4;
    const int i = token_of(kv, row0 + k, group);
    if (i > i_last) break;
    float M = -INFINITY, ls = 0.f, mw[CL * kAttnWarps];
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < CL * kAttnWarps; ++w) {
      const float* x = sm + (w % kAttnWarps * ROWS + k) * 2;
      if constexpr (CL > 1) x = cg::this_cluster().map_shared_rank(x, w / kAttnWarps);
      mw[w] = x[0];
      M = fmaxf(M, mw[w]);
    }
    const float zero = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < CL * kAttnWarps; ++w) {
      const float f = ex2(mw[w] - zero);
      const float* x = so + (w % kAttnWarps * ROWS + k) * LD + d;
      const float* y = sm + (w % kAttnWarps * ROWS + k) * 2 + 1;
      if constexpr (CL > 1) {
        x = cg::this_cluster().map_shared_rank(x, w / kAttnWarps);
        y = cg::this_cluster().map_shared_rank(y, w / kAttnWarps);
      }
      const float4 v = *reinterpret_cast<const float4*>(x);
      ls = fmaf(f, *y, ls);
      acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
    }
    if (CL > 1 || (first == 0 && last == n)) {
      const float inv = ls == 0.f ? 0.f : 1.f / ls;   // no key seen: zeros
      uint2 w;
      w.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      w.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(p.out + b * p.o_bstride + i * p.o_ld + (int64_t)(hk * group + row0 + k - i * group) * D + d) = w;
    } else {
      // a unit shared with other CTAs: a CTA has at most two, at its first block and at its last
      const int64_t pr = ((int64_t)blockIdx.x * 2 + (begins <= g0 ? 0 : 1)) * ROWS + k;
      *reinterpret_cast<float4*>(p.part_o + pr * D + d) = acc;
      if (d == 0) {
        p.part_ml[pr * 2] = M;
        p.part_ml[pr * 2 + 1] = ls;
      }
    }
  }
  if constexpr (CL > 1) {
    cg::this_cluster().sync();   // no CTA leaves while another reads its shared memory
    return;
  }
  // who has the first of a shared unit's blocks names it: the entry and head, and the CTAs that share it
  if (threadIdx.x == 0 && first == 0 && last < n)
    p.part_head[blockIdx.x] = make_int2(entry * kv.Hkv + hk, (begins + kSetup + n - 1) / per - (int)blockIdx.x + 1 + (begins <= g0 ? 0 : 1 << 30));
  g = begins + kSetup + last;
  if (g < g1) __syncthreads();   // the next unit stages its rows where the sums were
  }
}

// Joins a shared unit: one CTA per (CTA of the first kernel, row), exiting where that names none; each of its warps takes
// a quarter of the shares, D / 32 dims a lane.
template <int D>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Kv4AttnParams p) {
  constexpr int V = D / 32;
  __shared__ float part[4][D], sums[4];
  const Kv4Params& kv = p.kv;
  asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the first kernel runs
  const int2 head = p.part_head[blockIdx.x];
  if (head.x < 0) return;
  const int group = p.Hq / kv.Hkv, rows = 8 * p.row_nt, k = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int hk = head.x % kv.Hkv, entry = head.x / kv.Hkv, rt = entry % p.row_tiles, b = entry / p.row_tiles;
  const int R = rt * rows + k, i = token_of(kv, R, group);
  if (R >= kv.L * group || i >= new_tokens(kv, b)) return;
  // share s: slot 0 of the CTA blockIdx.x + s, but the first may be that CTA's slot 1
  const int shares = head.y & ((1 << 30) - 1);
  const auto slot = [&](int s) { return ((int64_t)(blockIdx.x + s) * 2 + (s == 0 ? head.y >> 30 : 0)) * rows + k; };
  float M = -INFINITY;
  for (int s = lane; s < shares; s += 32) M = fmaxf(M, p.part_ml[slot(s) * 2]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  const float z = M == -INFINITY ? 0.f : M;
  float l = 0.f, acc[V] = {};
#pragma unroll 4
  for (int s = warp; s < shares; s += 4) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot(s) * 2);
    const float f = ex2(ml.x - z);
    l = fmaf(f, ml.y, l);
    const float* src = p.part_o + slot(s) * D + lane * 2;
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      const float2 x = *reinterpret_cast<const float2*>(src + 32 * v);
      acc[v] = fmaf(f, x.x, acc[v]);
      acc[v + 1] = fmaf(f, x.y, acc[v + 1]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<float2*>(part[warp] + 32 * v + lane * 2) = make_float2(acc[v], acc[v + 1]);
  if (lane == 0) sums[warp] = l;
  __syncthreads();
  l = sums[0] + sums[1] + sums[2] + sums[3];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = p.out + b * p.o_bstride + i * p.o_ld + (int64_t)(hk * group + R - i * group) * D;
  for (int d = threadIdx.x; d < D; d += 128) dst[d] = __float2bfloat16_rn((part[0][d] + part[1][d] + part[2][d] + part[3][d]) * inv);
}

template <typename T>
cudaError_t launch_append_t(const Kv4AppendParams& p, unsigned rows, cudaStream_t stream) {
  const int hpw = 256 / p.kv.D;
  const int slots = (p.Hq + hpw - 1) / hpw + 2 * ((p.kv.Hkv + hpw - 1) / hpw);
  // with many tokens, fewer warps share a token's set-up (heads 32 + 2 x 8 of 128, 4 and 8 warps: 1 token 5.1 and 4.0 us,
  // 2048 tokens 19.0 and 18.4 us, 8000 tokens 49.8 and 55.9 us)
  const int threads = 32 * std::min(slots, rows >= 8u * device_sm_count() ? 4 : 8);
  switch (p.kv.D) {
    case 64: kv4_append_kernel<T, 64><<<rows, threads, 0, stream>>>(p); break;
    case 128: kv4_append_kernel<T, 128><<<rows, threads, 0, stream>>>(p); break;
    case 256: kv4_append_kernel<T, 256><<<rows, threads, 0, stream>>>(p); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4AppendParams& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.kv.B * p.kv.L;
  if (rows > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  return p.in_f32 ? launch_append_t<float>(p, (unsigned)rows, stream)
                  : launch_append_t<__nv_bfloat16>(p, (unsigned)rows, stream);
}

cudaError_t launch_kv4_read(const Kv4Params& p, __nv_bfloat16* out, int64_t ldo, int64_t bstride, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.B * p.L;
  if (rows > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  const int threads = std::min(256, (2 * p.Hkv * (p.D / 8) + 31) / 32 * 32);
  if (rows >= 8 * device_sm_count())   // one and two rows per CTA, 8 heads of 128: 1024 rows 3.4 and 3.7 us, 2048 5.2 and 4.9, 8000 17.2 and 15.3
    kv4_read_kernel<2><<<(unsigned)((rows + 1) / 2), threads, 0, stream>>>(p, out, ldo, bstride);
  else
    kv4_read_kernel<1><<<(unsigned)rows, threads, 0, stream>>>(p, out, ldo, bstride);
  return cudaGetLastError();
}

constexpr int kCluster = 8;

// Row tiles (two tiles of eight rows at a time share the converted operand where there are more than eight rows), and the
// CTAs: a cluster per unit where these fit one wave and no unit can be longer than eight blocks per warp (4096 tokens, by the
// page table's width or the window: lengths are on the device), else one wave, but at least a block of 16 tokens for each
// warp of the longest sequences.  Short sequences in a wide table therefore take the wave: 1024 tokens of D 256 in a table of
// 8192 10.4 us, in one of 1024 7.8.  Measured in us, 4 query heads per kv head:
//   cluster / wave            1 sequence of 1024: 7.5 / 9.8 (D 256), 6.3 / 8.4 (D 128);  16384: 27.2 / 29.7, 19.5 / 18.5;
//                             16 of 4096: 15.2 / 15.0, 11.2 / 12.6
//   16 rows, two tiles / one  2 x 32768 tokens, 8 kv heads of 128: 39.0 / 47.9;  12 rows: 37.7 / 47.4
//   4 rows, the low terms of P in the spare columns / in products of their own: 40 x 8192 tokens, 8 kv heads: 97.3 / 101.2
void kv4_attention_plan(Kv4AttnParams* p) {
  const Kv4Params& kv = p->kv;
  const int64_t rows = (int64_t)kv.L * (p->Hq / kv.Hkv);
  p->row_nt = rows > 8 ? 2 : 1;
  p->row_tiles = (int)((rows + 8 * p->row_nt - 1) / (8 * p->row_nt));
  const int64_t units = (int64_t)kv.B * kv.Hkv * p->row_tiles;
  const int64_t cap = (int64_t)kv.max_pages * kv.P / 16;
  const int64_t seen = p->window > 0 ? std::min(cap, ((int64_t)p->window + 8 * p->row_nt + 30) / 16 + ((int64_t)p->sinks + 15) / 16) : cap;
  int bits = 4;   // 2^bits tokens at least that a row may see
  while ((int64_t)1 << bits < seen * 16) ++bits;
  p->shift = bits + 1.f;
  const int wave = device_sm_count() * ctas_per_sm(kv.D, p->row_nt);
  p->cluster = units * kCluster <= wave && seen <= kCluster * kAttnWarps * 8;
  const int64_t most = (units * std::max<int64_t>(seen, 1) + kAttnWarps - 1) / kAttnWarps;
  p->ctas = p->cluster ? (int)units * kCluster : (int)std::min<int64_t>(most, wave);
}

// Blocks are counted in 32 bits.
bool kv4_attention_fits(Kv4AttnParams p) {
  const Kv4Params& kv = p.kv;
  const double tiles = (double)kv.B * kv.Hkv * (((double)kv.L * (p.Hq / kv.Hkv)) / 8 + 1);
  return tiles * ((double)kv.max_pages * kv.P / 16 + 1 + kSetup) < 2147480000.0;
}

// Two partial tiles per CTA (outputs, then maxima and sums), then the names of shared units.
size_t kv4_attention_workspace(Kv4AttnParams p) {
  kv4_attention_plan(&p);
  if (p.cluster) return 0;
  return (size_t)p.ctas * (2 * 8 * p.row_nt * (p.kv.D + 2) * 4 + 8);
}

namespace {

template <int D, int NT, bool SPLIT, int CL>
cudaError_t launch_attention_t(const Kv4AttnParams& p, cudaStream_t stream) {
  constexpr int bytes = (int)AttnSmem<D, NT>::bytes;
  if (bytes > 48 * 1024) {
    static DeviceOnce once;
    const cudaError_t e = once_per_device(
        once, [] { return cudaFuncSetAttribute(kv4_attention_kernel<D, NT, SPLIT, CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(kAttnWarps * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = CL;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_attention_kernel<D, NT, SPLIT, CL>, p);
  if (e != cudaSuccess || CL > 1 || p.ctas == 1) return e;
  cudaLaunchAttribute early;   // set up while the first kernel runs; it waits for that kernel's end by itself
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(p.ctas, 8 * NT);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D>, p);
}

template <int D, int CL>
cudaError_t launch_attention_r(const Kv4AttnParams& p, cudaStream_t stream) {
  if (p.kv.L * (p.Hq / p.kv.Hkv) <= 4) return launch_attention_t<D, 1, true, CL>(p, stream);
  return p.row_nt == 1 ? launch_attention_t<D, 1, false, CL>(p, stream) : launch_attention_t<D, 2, false, CL>(p, stream);
}

template <int D>
cudaError_t launch_attention_d(const Kv4AttnParams& p, cudaStream_t stream) {
  if (p.cluster)
    return launch_attention_r<D, kCluster>(p, stream);
  return launch_attention_r<D, 1>(p, stream);
}

}  // namespace

cudaError_t launch_kv4_attention(Kv4AttnParams p, void* workspace, cudaStream_t stream) {
  kv4_attention_plan(&p);
  if (!p.cluster) {
    const int64_t slots = (int64_t)p.ctas * 2 * 8 * p.row_nt;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + slots * p.kv.D;
    p.part_head = reinterpret_cast<int2*>(p.part_ml + slots * 2);
  }
  switch (p.kv.D) {
    case 64: return launch_attention_d<64>(p, stream);
    case 128: return launch_attention_d<128>(p, stream);
    case 256: return launch_attention_d<256>(p, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace nsa
