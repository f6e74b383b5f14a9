// The 4-bit paged key/value cache of a decode step (the format of q4.cuh, groups of 32 along the head
// dim): new tokens normalised, rotated and stored (append), stored tokens read back as bf16 rows, and
// attention over the cache.
//
// Pages: codes [n_pages][2][Hkv][P][D / 2] (keys, then values; value 2j in the low, 2j + 1 in the high
// nibble of byte j), scales [n_pages][2][Hkv][P][D / 32] bf16.  Token t of sequence b is slot t % P of page
// table[b][t / P].  A page id outside the pool, and a position outside the table (or the RoPE table), is
// recorded in the device error word and its access skipped.
#include <algorithm>

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

// Position of new token i of sequence b; -1 (recorded) when it lies outside the table.
__device__ __forceinline__ int position(const Kv4Params& p, int b, int i) {
  const int64_t pos = (int64_t)p.start[b] + i;
  if (p.start[b] < 0 || pos >= (int64_t)p.max_pages * p.P) {
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

// RMSNorm and rotation of one head held by LANES lanes: x[0..3] are elements 4 hl .. of the first half, x[4..7] their
// partners in the second; w the weights alike; c, s the cosines and sines of the four pairs.
template <typename T, int LANES>
__device__ __forceinline__ void norm_rope(const float* x, const float* w, const float* c, const float* s, bool rope, float eps,
                                          T* out) {
  T ss = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += (T)x[e] * (T)x[e];
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  T r;
  if constexpr (sizeof(T) == 8)
    r = rsqrt(ss * (1.0 / (8 * LANES)) + (double)eps);
  else
    r = rsqrtf(ss * (1.f / (8 * LANES)) + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = (T)x[e] * r * (T)w[e];
  if (rope) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const T a = out[e], b = out[4 + e];
      out[e] = a * (T)c[e] - b * (T)s[e];
      out[4 + e] = b * (T)c[e] + a * (T)s[e];
    }
  }
}

// A lane's four values of each half of a head's row of the cache (the group of 32 is eight lanes): even lanes store the
// pair's word of the first half, odd lanes that of the second.
template <bool SHORT, typename T>
__device__ __forceinline__ void store_codes(const T* x, uint8_t* codes, __nv_bfloat16* scales, int hl, int half, bool live) {
  float s[2];
  uint32_t bits[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float xf[4], am = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      xf[e] = (float)x[4 * k + e];
      am = amax2(fabsf(xf[e]), am);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) am = amax2(__shfl_xor_sync(0xffffffffu, am, o), am);
    s[k] = q4_scale(am);
    if constexpr (sizeof(T) == 8) {
      // fp64: where the rounded largest magnitude lies next to a border of two scales, the exact one decides (the
      // eight lanes of a group agree on it)
      const float below = __uint_as_float(__float_as_uint(s[k]) - 0x00080000u), near = am * 0x1p-22f;
      if (fabsf(7.f * s[k] - am) <= near || fabsf(7.f * below - am) <= near || fabsf(am - 0x1p-110f) <= near || !isfinite(am)) {
        const unsigned lanes = 0xFFu << (threadIdx.x & 24);
        double exact = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) exact = amax2(fabs((double)x[4 * k + e]), exact);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) exact = amax2(__shfl_xor_sync(lanes, exact, o), exact);
        s[k] = q4_scale(exact);
      }
    }
    bits[k] = s[k] > 0.f ? q4_bits<4, q4_in_order, SHORT>(x + 4 * k, xf, s[k], am) : 0x8888u;
  }
  const bool odd = hl & 1;
  const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? bits[0] : bits[1], 1);
  if (!live) return;
  const uint32_t word = odd ? got | (bits[1] << 16) : bits[0] | (got << 16);
  *reinterpret_cast<uint32_t*>(codes + (odd ? half / 2 : 0) + hl / 2 * 4) = word;
  if (hl % 8 < 2) scales[(odd ? half / kKvGroup : 0) + hl / 8] = __float2bfloat16_rn(odd ? s[1] : s[0]);
}

// A CTA per token; a warp takes 256 / D heads of one kind (q, k or v) at a time, eight values a lane.  Bound by the
// bytes of q | k | v.  Keys are computed in fp64: the code of a value next to the border of two codes is
// decided by the last bits, and the fp32 order of sums would decide it by chance.
template <typename T, int D>
__global__ void __launch_bounds__(256, 3) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int LANES = D / 8, HPW = 32 / LANES, half = D / 2;
  const Kv4Params& kv = p.kv;
  const int lane = threadIdx.x % 32, hl = lane % LANES;
  const int q_slots = (p.Hq + HPW - 1) / HPW, kv_slots = (kv.Hkv + HPW - 1) / HPW;
  const int b = blockIdx.x / kv.L, i = blockIdx.x % kv.L;
  if (i >= new_tokens(kv, b)) return;
  const int pos = position(kv, b, i);
  if (pos < 0) return;
  if (p.cs && pos >= p.rope_rows) {
    if (threadIdx.x == 0) atomicCAS(kv.err, 0, kErrKvPosition);
    return;
  }
  const T* row = static_cast<const T*>(p.qkv) + b * p.bstride + i * p.ld;
  for (int slot = threadIdx.x / 32; slot < q_slots + 2 * kv_slots; slot += blockDim.x / 32) {
    const int kind = slot < q_slots ? 0 : slot < q_slots + kv_slots ? 1 : 2;
    const int heads = kind == 0 ? p.Hq : kv.Hkv;
    const int h = (kind == 0 ? slot : slot - q_slots - (kind - 1) * kv_slots) * HPW + lane / LANES;
    const bool live = h < heads;                                   // lanes past the last head repeat it, storing nothing
    const int hh = live ? h : heads - 1;
    const T* src = row + (kind == 0 ? p.q_off : kind == 1 ? p.k_off : p.v_off) + (int64_t)hh * D + hl * 4;
    float x[8], w[8], c[4], s[4];
    load4(src, x);
    load4(src + half, x + 4);
    if (kind < 2) {
      const float* wt = (kind == 0 ? p.q_w : p.k_w) + hl * 4;
      load4(wt, w);
      load4(wt + half, w + 4);
      if (p.cs) {
        const float* t = p.cs + (int64_t)pos * half + hl * 4;
        load4(t, c);
        load4(t + p.sin_off, s);
      }
    }
    if (kind == 0) {
      float o[8];
      norm_rope<float, LANES>(x, w, c, s, p.cs != nullptr, p.eps, o);
      if (live) {
        __nv_bfloat16* dst = p.q_out + b * p.qo_bstride + i * p.qo_ld + (int64_t)hh * D + hl * 4;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
        *reinterpret_cast<uint2*>(dst + half) = make_uint2(pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
      }
      continue;
    }
    const int page = page_of(kv, b, pos);
    if (page < 0) return;
    const int64_t tok = cache_row(kv, page, kind - 1, hh, pos);
    uint8_t* codes = kv.codes + tok * (D / 2);
    __nv_bfloat16* scales = kv.scales + tok * (D / kKvGroup);
    if (kind == 1) {
      double o[8];
      norm_rope<double, LANES>(x, w, c, s, p.cs != nullptr, p.eps, o);
      store_codes<false>(o, codes, scales, hl, half, live);
    } else {
      store_codes<sizeof(T) == 2>(x, codes, scales, hl, half, live);
    }
  }
}

// A CTA per row, a thread per word (8 values).
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Params p, __nv_bfloat16* __restrict__ out, int64_t ldo,
                                                       int64_t bstride) {
  const int b = blockIdx.x / p.L, i = blockIdx.x % p.L;
  if (i >= new_tokens(p, b)) return;
  const int pos = position(p, b, i);
  if (pos < 0) return;
  const int page = page_of(p, b, pos);
  if (page < 0) return;
  const int words = p.D / 8;
  for (int e = threadIdx.x; e < 2 * p.Hkv * words; e += blockDim.x) {
    const int w = e % words, h = e / words;                        // h: key heads, then value heads
    const int64_t tok = cache_row(p, page, 0, h, pos);             // heads of both halves follow one another
    const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(p.codes + tok * (p.D / 2)) + w);
    const uint16_t sc = __ldg(reinterpret_cast<const uint16_t*>(p.scales) + tok * (p.D / kKvGroup) + w * 8 / kKvGroup);
    uint32_t s2;
    asm("mov.b32 %0, {%1, %1};" : "=r"(s2) : "h"(sc));
    const uint32_t v04 = mul_bf16x2(code_pair<0>(v), s2), v15 = mul_bf16x2(code_pair<1>(v), s2);
    const uint32_t v26 = mul_bf16x2(code_pair<2>(v), s2), v37 = mul_bf16x2(code_pair<3>(v), s2);
    uint4 o;
    o.x = __byte_perm(v04, v15, 0x5410);
    o.y = __byte_perm(v26, v37, 0x5410);
    o.z = __byte_perm(v04, v15, 0x7632);
    o.w = __byte_perm(v26, v37, 0x7632);
    reinterpret_cast<uint4*>(out + b * bstride + i * ldo)[e] = o;
  }
}

// ------------------------------------------------------------------------------------ attention
//
// A CTA takes eight query rows that share a key/value head (row R of sequence b is new token R / group, query
// head R % group of the head's group) and a share of the keys; each of its warps walks its own blocks of 16
// tokens (a block never straddles pages) with its own running maximum, sum and output, joined in shared memory
// at the end and, when the keys are split over CTAs, by a second kernel.
//
// Both products run on mma.m16n8k16 with the cached operand as A, so that the eight query rows fill N = 8 and
// only the cache's bytes are converted:
//   S^T [16 tokens][8 rows] = K [16 tokens][D] Q^T,   O^T [D][8 rows] += V^T [D][16 tokens] P^T.
// A tcgen05 tile would need the converted operand in shared memory (4 times the cache's bytes written and
// read again there); here each lane loads 4-bit words straight from global memory in the A fragment's own
// order, converts them in registers and multiplies.  The contraction index of a product may be permuted, so
// lane (r, c) = (lane / 4, lane % 4) takes, of token r, the 16-byte pieces c of the row: nibbles p and p + 4
// of a word are one bf16 pair, and Q is staged in the matching order.  For V the lane takes piece r of the
// tokens 2c, 2c + 1, 2c + 8, 2c + 9 (what its B fragment of P^T holds) and pairs the tokens' words by byte
// permutes; the rows of an output tile are the lane's own dims.  Conversion: a nibble n moved to the top of a
// bf16 mantissa is 1 + n / 16, and (1 + n / 16) 16 s - 24 s = s (n - 8) is one bf16x2 fma, exact because the
// scale has five significant bits (q4.cuh).
//
// P^T is P's accumulator transposed: packed to bf16 and turned by movmatrix.  P is split into two bf16 terms
// (16 bits together): one bf16 would add an error as large as the output's own rounding.
// The running maximum moves only when a score exceeds it by 2^8 in the exponent's base, which keeps sums in
// range without a reduction over lanes per block.

constexpr int kAttnWarps = 4;
constexpr float kMaxSlack = 8.f;   // exp2 of a score may reach 2^8 before the maximum is moved

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
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
  return fma_bf16x2((m & 0x00780078u) | 0x3F803F80u, s.s16, s.m24);
}

// N 32-bit words (1, 2 or 4 aligned, 8 as two pieces 64 bytes apart).
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* src, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(src));
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
    w[0] = v.x; w[1] = v.y;
  } else if constexpr (N == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
    load_words<4>(src, w);
    load_words<4>(src + 64, w + 4);
  }
}

// Which 16-token blocks the rows of a tile see: [0, sink_blocks), then from first on; n in all.
struct Blocks {
  int sink_blocks, first, n;
};
__device__ __forceinline__ Blocks blocks_of(int pmin, int pmax, int window, int sinks) {
  if (pmax < 0) return {0, 0, 0};
  const int lo = window > 0 ? max(0, pmin - window + 1) : 0;
  const int first = lo / 16;
  const int ns = min((min(sinks, lo) + 15) / 16, first);
  return {ns, first, ns + pmax / 16 - first + 1};
}

template <int D>
struct AttnSmem {
  static constexpr size_t q = (size_t)D / 16 * 32 * 8;                       // Q^T fragments
  static constexpr size_t o = (size_t)kAttnWarps * 8 * (D + 4) * 4;          // warps' outputs, rows padded
  static constexpr size_t bytes = (q > o ? q : o) + kAttnWarps * 8 * 2 * 4;  // ... and their (m, l); below 48 KB
};

template <int D>
__global__ void __launch_bounds__(kAttnWarps * 32, D == 256 ? 3 : 4) kv4_attention_kernel(const Kv4AttnParams p) {
  constexpr int KW = D / 32;   // words of a token's keys per lane
  constexpr int VW = D / 64;   // words of a token's values per lane
  constexpr int KG = D == 256 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  const Kv4Params& kv = p.kv;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
  const int group = p.Hq / kv.Hkv;
  const int split = blockIdx.x % p.splits;
  int u = blockIdx.x / p.splits;
  const int unit = u;
  const int rt = u % p.row_tiles;
  u /= p.row_tiles;
  const int hk = u % kv.Hkv, b = u / kv.Hkv;
  const int rows = min(8, kv.L * group - rt * 8);
  const int cnt = new_tokens(kv, b);
  // positions of the tile's rows (-1: not a row of this step, or outside the table)
  int pos0 = -1, pos1 = -1, pmin = 0x7FFFFFFF, pmax = -1;
  bool outside = false;
  for (int k = 0; k < rows; ++k) {
    const int i = (rt * 8 + k) / group;
    if (i >= cnt) break;
    const int pos = position(kv, b, i);
    if (pos >= 0) pmin = min(pmin, pos);
    else outside = true;
    pmax = max(pmax, pos);
    if (k == 2 * c) pos0 = pos;
    if (k == 2 * c + 1) pos1 = pos;
  }
  const Blocks bl = blocks_of(pmin, pmax, p.window, p.sinks);
  const int share = (bl.n + p.splits - 1) / p.splits;
  const int t1 = min(bl.n, (split + 1) * share);
  int t = split * share + warp;

  // Q^T fragments: for k-step 2w + s of lane (r, c), words of row r's dims in the order of the lane's key words
  uint2* qs = reinterpret_cast<uint2*>(smem);
  for (int e = threadIdx.x; e < D / 16 * 32; e += kAttnWarps * 32) {
    const int ks = e / 32, ln = e % 32, rr = ln / 4, cc = ln % 4, w = ks / 2, s2 = ks % 2;
    const int word = D == 256 ? 4 * (cc + 4 * (w / 4)) + w % 4 : KW * cc + w;
    uint2 f = make_uint2(0u, 0u);
    const int i = (rt * 8 + rr) / group;
    if (rr < rows && i < cnt) {
      const uint4 v = *reinterpret_cast<const uint4*>(p.q + b * p.q_bstride + i * p.q_ld +
                                                      (int64_t)(hk * group + (rt * 8 + rr) % group) * D + word * 8);
      // pairs (e, e + 4): e = 2 s2 and 2 s2 + 1
      const uint32_t lo = s2 ? v.y : v.x, hi = s2 ? v.w : v.z;
      f = make_uint2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
    }
    qs[e] = f;
  }
  __syncthreads();

  float o[VW * 4][4];
#pragma unroll
  for (int x = 0; x < VW * 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) o[x][y] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, z0 = 0.f, z1 = 0.f, l0 = 0.f, l1 = 0.f;   // z: the maximum subtracted (0 while none)

  uint32_t kw[2][KW], vw[4][VW];
  uint32_t ks[2][KG], vs[4];
  const int* table = kv.table + (int64_t)b * kv.table_ld;
  const int64_t head = (int64_t)hk * kv.P, page_rows = (int64_t)2 * kv.Hkv * kv.P;
  const auto block_at = [&](int tt) { return tt < bl.sink_blocks ? tt : bl.first + tt - bl.sink_blocks; };
  // row of the block's first token in the key half of its page, or -1
  const auto row_of = [&](int tt) -> int64_t {
    if (tt >= t1) return -1;
    const int j = block_at(tt) * 16;
    const int id = __ldg(table + j / kv.P);
    if (id < 0 || id >= kv.n_pages) {
      if (lane == 0) atomicCAS(kv.err, 0, kErrKvPage);
      return -1;
    }
    return id * page_rows + head + j % kv.P;
  };
  const auto load_k = [&](int64_t row) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (row < 0) {
#pragma unroll
        for (int y = 0; y < KW; ++y) kw[x][y] = 0;
#pragma unroll
        for (int y = 0; y < KG; ++y) ks[x][y] = 0;
        continue;
      }
      const int64_t tok = row + r + 8 * x;
      load_words<KW>(kv.codes + tok * (D / 2) + (D == 256 ? 16 : KW * 4) * c, kw[x]);
      const uint16_t* sc = reinterpret_cast<const uint16_t*>(kv.scales) + tok * (D / 32);
#pragma unroll
      for (int y = 0; y < KG; ++y) ks[x][y] = __ldg(sc + (D == 64 ? c / 2 : c + 4 * y));
    }
  };
  const auto load_v = [&](int64_t row) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (row < 0) {
#pragma unroll
        for (int y = 0; y < VW; ++y) vw[x][y] = 0;
        vs[x] = 0;
        continue;
      }
      const int64_t tok = row + (int64_t)kv.Hkv * kv.P + 2 * c + (x & 1) + 8 * (x >> 1);
      load_words<VW>(kv.codes + tok * (D / 2) + VW * 4 * r, vw[x]);
      vs[x] = __ldg(reinterpret_cast<const uint16_t*>(kv.scales) + tok * (D / 32) + r * VW / 4);
    }
  };

  int64_t row = row_of(t);
  if (t < t1) {
    load_k(row);
    load_v(row);
  }
  int64_t next = row_of(t + kAttnWarps);
  for (; t < t1; t += kAttnWarps) {
    float s[2][4] = {};
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const int g = KG == 2 ? w / 4 : 0;
      const ScalePair sa = scale_pair(ks[0][g], ks[0][g]), sb = scale_pair(ks[1][g], ks[1][g]);
      const uint2 q0 = qs[(2 * w) * 32 + lane], q1 = qs[(2 * w + 1) * 32 + lane];
      mma_bf16(s[0], dequant<0>(kw[0][w], sa), dequant<0>(kw[1][w], sb), dequant<1>(kw[0][w], sa), dequant<1>(kw[1][w], sb), q0.x, q0.y);
      mma_bf16(s[1], dequant<2>(kw[0][w], sa), dequant<2>(kw[1][w], sb), dequant<3>(kw[0][w], sa), dequant<3>(kw[1][w], sb), q1.x, q1.y);
    }
    const int j0 = block_at(t) * 16;
    const bool missing = row < 0;
    if (t + kAttnWarps < t1) load_k(next);
    float x0 = (s[0][0] + s[1][0]) * p.scale_log2, x1 = (s[0][1] + s[1][1]) * p.scale_log2;
    float x2 = (s[0][2] + s[1][2]) * p.scale_log2, x3 = (s[0][3] + s[1][3]) * p.scale_log2;
    const bool whole = !missing && !outside && j0 + 15 <= pmin && (p.window == 0 || j0 > pmax - p.window || j0 + 15 < p.sinks);
    if (!whole) {
      const auto see = [&](int pos, int j) {
        return !missing && j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks);
      };
      if (!see(pos0, j0 + r)) x0 = -INFINITY;
      if (!see(pos1, j0 + r)) x1 = -INFINITY;
      if (!see(pos0, j0 + r + 8)) x2 = -INFINITY;
      if (!see(pos1, j0 + r + 8)) x3 = -INFINITY;
      // tokens no row sees may hold anything: their values become zeros
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int j = j0 + 2 * c + (x & 1) + 8 * (x >> 1);
        if (missing || j > pmax || (p.window > 0 && j <= pmin - p.window && j >= p.sinks)) vs[x] = 0;
      }
    }
    const bool up = x0 > m0 + kMaxSlack || x2 > m0 + kMaxSlack || x1 > m1 + kMaxSlack || x3 > m1 + kMaxSlack;
    if (__any_sync(0xffffffffu, up)) {
      float n0 = fmaxf(x0, x2), n1 = fmaxf(x1, x3);
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, d));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, d));
      }
      n0 = fmaxf(n0, m0);
      n1 = fmaxf(n1, m1);
      const float y0 = n0 == -INFINITY ? 0.f : n0, y1 = n1 == -INFINITY ? 0.f : n1;
      const float f0 = exp2f(m0 - y0), f1 = exp2f(m1 - y1);
      m0 = n0; m1 = n1; z0 = y0; z1 = y1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int x = 0; x < VW * 4; ++x) {
        o[x][0] *= f0; o[x][1] *= f1;
        o[x][2] *= f0; o[x][3] *= f1;
      }
    }
    x0 = exp2f(x0 - z0); x1 = exp2f(x1 - z1);
    x2 = exp2f(x2 - z0); x3 = exp2f(x3 - z1);
    l0 += x0 + x2;
    l1 += x1 + x3;
    const uint32_t h0 = pack_bf16x2(x0, x1), h1 = pack_bf16x2(x2, x3);
    const uint32_t e0 = pack_bf16x2(x0 - __uint_as_float(h0 << 16), x1 - __uint_as_float(h0 & 0xFFFF0000u));
    const uint32_t e1 = pack_bf16x2(x2 - __uint_as_float(h1 << 16), x3 - __uint_as_float(h1 & 0xFFFF0000u));
    const uint32_t ph0 = transpose8x8(h0), ph1 = transpose8x8(h1), pl0 = transpose8x8(e0), pl1 = transpose8x8(e1);
    // A value group with an infinity or a NaN is NaN in the outputs of the rows that see it; as a factor it
    // would reach the others too (0 * NaN), so it leaves the product and is added to its rows here.
    bool odd = false;
#pragma unroll
    for (int x = 0; x < 4; ++x) odd |= (vs[x] & 0x7F80u) == 0x7F80u;
    if (__any_sync(0xffffffffu, odd)) {
      for (int k = 0; k < 16; ++k) {
        const int x = (k & 1) + 2 * (k >> 3), src = r * 4 + (k % 8) / 2;
        const uint32_t sk = __shfl_sync(0xffffffffu, x == 0 ? vs[0] : x == 1 ? vs[1] : x == 2 ? vs[2] : vs[3], src);
        if ((sk & 0x7F80u) != 0x7F80u) continue;
        const int j = j0 + k;
        const auto see = [&](int pos) { return j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks); };
        const float nan = __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int y = 0; y < VW * 4; ++y) {
          if (see(pos0)) o[y][0] = nan, o[y][2] = nan;
          if (see(pos1)) o[y][1] = nan, o[y][3] = nan;
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if ((vs[x] & 0x7F80u) == 0x7F80u) vs[x] = 0;
    }
    const ScalePair va = scale_pair(vs[0], vs[1]), vb = scale_pair(vs[2], vs[3]);
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const uint32_t xa = __byte_perm(vw[0][w], vw[1][w], 0x5410), ya = __byte_perm(vw[0][w], vw[1][w], 0x7632);
      const uint32_t xb = __byte_perm(vw[2][w], vw[3][w], 0x5410), yb = __byte_perm(vw[2][w], vw[3][w], 0x7632);
      const auto tile = [&](float* acc, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
        mma_bf16(acc, a0, a1, a2, a3, ph0, ph1);
        mma_bf16(acc, a0, a1, a2, a3, pl0, pl1);
      };
      tile(o[4 * w + 0], dequant<0>(xa, va), dequant<0>(ya, va), dequant<0>(xb, vb), dequant<0>(yb, vb));
      tile(o[4 * w + 1], dequant<1>(xa, va), dequant<1>(ya, va), dequant<1>(xb, vb), dequant<1>(yb, vb));
      tile(o[4 * w + 2], dequant<2>(xa, va), dequant<2>(ya, va), dequant<2>(xb, vb), dequant<2>(yb, vb));
      tile(o[4 * w + 3], dequant<3>(xa, va), dequant<3>(ya, va), dequant<3>(xb, vb), dequant<3>(yb, vb));
    }
    if (t + kAttnWarps < t1) load_v(next);
    row = next;
    next = row_of(t + 2 * kAttnWarps);
  }
#pragma unroll
  for (int d = 4; d < 32; d <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, d);
    l1 += __shfl_xor_sync(0xffffffffu, l1, d);
  }

  // join the warps
  __syncthreads();   // the fragments of Q are no longer read
  float* so = reinterpret_cast<float*>(smem);
  float* sm = reinterpret_cast<float*>(smem + AttnSmem<D>::bytes - kAttnWarps * 8 * 2 * 4);
  constexpr int LD = D + 4;
#pragma unroll
  for (int w = 0; w < VW; ++w)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = 8 * (VW * r + w) + x;
      float* row0 = so + (warp * 8 + 2 * c) * LD + d;
      row0[0] = o[4 * w + x][0];
      row0[LD] = o[4 * w + x][1];
      row0[4] = o[4 * w + x][2];
      row0[LD + 4] = o[4 * w + x][3];
    }
  if (r == 0) {
    float* ml = sm + (warp * 8 + 2 * c) * 2;
    ml[0] = m0; ml[1] = l0;
    ml[2] = m1; ml[3] = l1;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * (D / 4); e += kAttnWarps * 32) {
    const int k = e / (D / 4), d = e % (D / 4) * 4;
    const int i = (rt * 8 + k) / group;
    if (i >= cnt) break;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) M = fmaxf(M, sm[(w * 8 + k) * 2]);
    const float z = M == -INFINITY ? 0.f : M;
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f = exp2f(sm[(w * 8 + k) * 2] - z);
      const float4 v = *reinterpret_cast<const float4*>(so + (w * 8 + k) * LD + d);
      l = fmaf(f, sm[(w * 8 + k) * 2 + 1], l);
      acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
    }
    if (p.splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;   // no key seen: zeros
      uint2 w;
      w.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      w.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(p.out + b * p.o_bstride + i * p.o_ld + (int64_t)(hk * group + (rt * 8 + k) % group) * D + d) = w;
    } else {
      const int64_t pr = ((int64_t)unit * p.splits + split) * 8 + k;
      *reinterpret_cast<float4*>(p.part_o + pr * D + d) = acc;
      if (d == 0) {
        p.part_ml[pr * 2] = M;
        p.part_ml[pr * 2 + 1] = l;
      }
    }
  }
}

// Joins the shares of a row's keys: one CTA per (unit, row), a thread per dim.
__global__ void kv4_join_kernel(const Kv4AttnParams p) {
  const Kv4Params& kv = p.kv;
  const int D = kv.D, group = p.Hq / kv.Hkv;
  const int k = blockIdx.x % 8;
  const int64_t unit = blockIdx.x / 8;
  const int rt = (int)(unit % p.row_tiles), hk = (int)(unit / p.row_tiles % kv.Hkv), b = (int)(unit / p.row_tiles / kv.Hkv);
  const int R = rt * 8 + k, i = R / group;
  if (R >= kv.L * group || i >= new_tokens(kv, b)) return;
  const int64_t pr = unit * p.splits * 8 + k;
  float M = -INFINITY;
  for (int s = 0; s < p.splits; ++s) M = fmaxf(M, p.part_ml[(pr + s * 8) * 2]);
  const float z = M == -INFINITY ? 0.f : M;
  float l = 0.f, acc = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float f = exp2f(p.part_ml[(pr + s * 8) * 2] - z);
    l = fmaf(f, p.part_ml[(pr + s * 8) * 2 + 1], l);
    acc = fmaf(f, p.part_o[(pr + s * 8) * D + threadIdx.x], acc);
  }
  p.out[b * p.o_bstride + i * p.o_ld + (int64_t)(hk * group + R % group) * D + threadIdx.x] =
      __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
}

template <typename T>
cudaError_t launch_append_t(const Kv4AppendParams& p, unsigned rows, cudaStream_t stream) {
  const int hpw = 256 / p.kv.D;
  const int slots = (p.Hq + hpw - 1) / hpw + 2 * ((p.kv.Hkv + hpw - 1) / hpw);
  const int threads = 32 * std::min(slots, 8);
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
  kv4_read_kernel<<<(unsigned)rows, threads, 0, stream>>>(p, out, ldo, bstride);
  return cudaGetLastError();
}

constexpr int kCtasWanted = 4 * 3 * 148;   // four waves of three CTAs on each of a B200's SMs

// Row tiles, and how many CTAs share a tile's keys: enough for a few CTAs per SM and to even out sequences of
// different lengths, as long as each warp keeps two blocks of 16 tokens of the longest sequence.
void kv4_attention_plan(Kv4AttnParams* p) {
  const Kv4Params& kv = p->kv;
  p->row_tiles = (int)(((int64_t)kv.L * (p->Hq / kv.Hkv) + 7) / 8);
  const int64_t units = (int64_t)kv.B * kv.Hkv * p->row_tiles;
  const int64_t cap = (int64_t)kv.max_pages * kv.P;
  const int64_t seen = p->window > 0 ? std::min(cap, (int64_t)p->window + p->sinks + kv.L + 30) : cap;
  const int64_t want = (kCtasWanted + units - 1) / units;
  const int64_t most = (seen + 16 * kAttnWarps * 2 - 1) / (16 * kAttnWarps * 2);
  p->splits = (int)std::max<int64_t>(1, std::min(want, most));
}

size_t kv4_attention_workspace(Kv4AttnParams p) {
  kv4_attention_plan(&p);
  if (p.splits == 1) return 0;
  return (size_t)p.kv.B * p.kv.Hkv * p.row_tiles * p.splits * 8 * (p.kv.D + 2) * 4;
}

namespace {

template <int D>
cudaError_t launch_attention_t(const Kv4AttnParams& p, unsigned blocks, cudaStream_t stream) {
  kv4_attention_kernel<D><<<blocks, kAttnWarps * 32, AttnSmem<D>::bytes, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_attention(Kv4AttnParams p, void* workspace, cudaStream_t stream) {
  kv4_attention_plan(&p);
  const int64_t units = (int64_t)p.kv.B * p.kv.Hkv * p.row_tiles;
  if (units * p.splits > 0x7FFFFFFFLL || units * 8 > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + units * p.splits * 8 * p.kv.D;
  const unsigned blocks = (unsigned)(units * p.splits);
  cudaError_t e;
  switch (p.kv.D) {
    case 64: e = launch_attention_t<64>(p, blocks, stream); break;
    case 128: e = launch_attention_t<128>(p, blocks, stream); break;
    case 256: e = launch_attention_t<256>(p, blocks, stream); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess || p.splits == 1) return e;
  kv4_join_kernel<<<(unsigned)(units * 8), p.kv.D, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace nsa
