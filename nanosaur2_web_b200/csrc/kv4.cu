// The 4-bit paged key/value cache of a decode step (the format of q4.cuh, groups of 32 along the head
// dim): new tokens normalised, rotated and stored (append), stored tokens read back as bf16 rows, and
// attention over the cache.
//
// Pages: codes [n_pages][2][Hkv][P][D / 2] (keys, then values; value 2j in the low, 2j + 1 in the high
// nibble of byte j), scales [n_pages][2][Hkv][P][D / 32] bf16.  Token t of sequence b is slot t % P of page
// table[b][t / P].  A page id outside the pool, and a position outside the table (or the RoPE table), is
// recorded in the device error word and its access skipped.
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

// N (1, 2 or 4) consecutive inputs.
template <int N>
__device__ __forceinline__ void load_n(const float* src, float* x) {
  if constexpr (N == 4) {
    const float4 v = *reinterpret_cast<const float4*>(src);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else if constexpr (N == 2) {
    const float2 v = *reinterpret_cast<const float2*>(src);
    x[0] = v.x; x[1] = v.y;
  } else {
    x[0] = *src;
  }
}
template <int N>
__device__ __forceinline__ void load_n(const __nv_bfloat16* src, float* x) {
  if constexpr (N == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xFFFF0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xFFFF0000u);
  } else if constexpr (N == 2) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(src);
    x[0] = __uint_as_float(v << 16); x[1] = __uint_as_float(v & 0xFFFF0000u);
  } else {
    x[0] = __bfloat162float(*src);
  }
}

template <typename T>
__device__ __forceinline__ T warp_sum_t(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// RMSNorm times w and the rotation of pairs (i, i + D/2) of one head held by a warp: a[j], b[j] are
// elements i = lane * HN + j and D/2 + i.
template <typename T, int HN>
__device__ __forceinline__ void norm_rope(T* a, T* b, const Kv4AppendParams& p, const float* w, int pos, int lane) {
  constexpr int half = 32 * HN;
  T ss = 0;
#pragma unroll
  for (int j = 0; j < HN; ++j) ss += a[j] * a[j] + b[j] * b[j];
  ss = warp_sum_t(ss);
  T r;
  if constexpr (sizeof(T) == 8)
    r = 1.0 / sqrt(ss / (2 * half) + (double)p.eps);
  else
    r = rsqrtf(ss / (float)(2 * half) + p.eps);
  float wa[HN], wb[HN], c[HN], s[HN];
  load_n<HN>(w + lane * HN, wa);
  load_n<HN>(w + half + lane * HN, wb);
  if (p.cs) {
    load_n<HN>(p.cs + (int64_t)pos * half + lane * HN, c);
    load_n<HN>(p.cs + p.sin_off + (int64_t)pos * half + lane * HN, s);
  }
#pragma unroll
  for (int j = 0; j < HN; ++j) {
    const T y1 = a[j] * r * (T)wa[j], y2 = b[j] * r * (T)wb[j];
    a[j] = p.cs ? y1 * (T)c[j] - y2 * (T)s[j] : y1;
    b[j] = p.cs ? y2 * (T)c[j] + y1 * (T)s[j] : y2;
  }
}

// HN consecutive elements per lane, one half of a head: scale over the 32 / HN lanes of a group, codes
// packed into bytes and stored at dst (this half's codes), scales at sc.
template <typename T, int HN>
__device__ __forceinline__ void store_half(const T* x, uint8_t* dst, __nv_bfloat16* sc, int lane) {
  T am = 0;
#pragma unroll
  for (int j = 0; j < HN; ++j) am = amax2(fabs(x[j]), am);
#pragma unroll
  for (int o = 1; o < 32 / HN; o <<= 1) am = amax2(__shfl_xor_sync(0xffffffffu, am, o), am);
  const float s = q4_scale(am);
  uint32_t bits = 0x8888u >> (16 - 4 * HN);
  if (s > 0.f) {
    const T inv = (T)1 / (T)s;
    bits = 0;
#pragma unroll
    for (int j = 0; j < HN; ++j) bits |= q4_code(x[j], (T)s, inv) << (4 * j);
  }
  if constexpr (HN == 4) {
    reinterpret_cast<uint16_t*>(dst)[lane] = (uint16_t)bits;
  } else if constexpr (HN == 2) {
    dst[lane] = (uint8_t)bits;
  } else {
    const uint32_t up = __shfl_down_sync(0xffffffffu, bits, 1);
    if (lane % 2 == 0) dst[lane / 2] = (uint8_t)(bits | (up << 4));
  }
  if (lane % (32 / HN) == 0) sc[lane / (32 / HN)] = __float2bfloat16_rn(s);
}

// One warp per (token, head) of q | k | v.  Keys are computed in fp64: the code of a value next to the
// border of two codes is decided by the last bits, and the fp32 order of sums would decide it by chance.
template <typename T, int HN>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int D = 64 * HN, half = D / 2;
  const Kv4Params& kv = p.kv;
  const int lane = threadIdx.x % 32;
  const int heads = p.Hq + 2 * kv.Hkv;
  const int64_t unit = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (unit >= (int64_t)kv.B * kv.L * heads) return;
  const int h = (int)(unit % heads);
  const int64_t row = unit / heads;
  const int b = (int)(row / kv.L), i = (int)(row % kv.L);
  if (i >= new_tokens(kv, b)) return;
  const int pos = position(kv, b, i);
  if (pos < 0) return;
  if (p.cs && pos >= p.rope_rows) {
    if (lane == 0) atomicCAS(kv.err, 0, kErrKvPosition);
    return;
  }
  const bool is_q = h < p.Hq, is_k = !is_q && h < p.Hq + kv.Hkv;
  const int hh = is_q ? h : (is_k ? h - p.Hq : h - p.Hq - kv.Hkv);
  const int64_t off = is_q ? p.q_off : (is_k ? p.k_off : p.v_off);
  const T* src = static_cast<const T*>(p.qkv) + b * p.bstride + i * p.ld + off + (int64_t)hh * D;
  float a[HN], c[HN];
  load_n<HN>(src + lane * HN, a);
  load_n<HN>(src + half + lane * HN, c);
  if (is_q) {
    norm_rope<float, HN>(a, c, p, p.q_w, pos, lane);
    __nv_bfloat16* dst = p.q_out + b * p.qo_bstride + i * p.qo_ld + (int64_t)hh * D;
#pragma unroll
    for (int j = 0; j < HN; ++j) {
      dst[lane * HN + j] = __float2bfloat16_rn(a[j]);
      dst[half + lane * HN + j] = __float2bfloat16_rn(c[j]);
    }
    return;
  }
  const int page = page_of(kv, b, pos);
  if (page < 0) return;
  const int64_t tok = cache_row(kv, page, is_k ? 0 : 1, hh, pos);
  uint8_t* codes = kv.codes + tok * (D / 2);
  __nv_bfloat16* scales = kv.scales + tok * (D / kKvGroup);
  if (is_k) {
    double ad[HN], cd[HN];
#pragma unroll
    for (int j = 0; j < HN; ++j) ad[j] = a[j], cd[j] = c[j];
    norm_rope<double, HN>(ad, cd, p, p.k_w, pos, lane);
    store_half<double, HN>(ad, codes, scales, lane);
    store_half<double, HN>(cd, codes + half / 2, scales + half / kKvGroup, lane);
  } else {
    store_half<float, HN>(a, codes, scales, lane);
    store_half<float, HN>(c, codes + half / 2, scales + half / kKvGroup, lane);
  }
}

// One thread per word (8 values) of a read-back row.
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Params p, __nv_bfloat16* __restrict__ out, int64_t ldo,
                                                       int64_t bstride) {
  const int words = p.D / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int w = (int)(idx % words);
  int64_t r = idx / words;
  const int h = (int)(r % p.Hkv);
  r /= p.Hkv;
  const int which = (int)(r % 2);
  r /= 2;
  const int i = (int)(r % p.L);
  const int64_t b = r / p.L;
  if (b >= p.B || i >= new_tokens(p, (int)b)) return;
  const int pos = position(p, (int)b, i);
  if (pos < 0) return;
  const int page = page_of(p, (int)b, pos);
  if (page < 0) return;
  const int64_t tok = cache_row(p, page, which, h, pos);
  const uint32_t v = reinterpret_cast<const uint32_t*>(p.codes + tok * (p.D / 2))[w];
  const float s = __bfloat162float(p.scales[tok * (p.D / kKvGroup) + w * 8 / kKvGroup]);
  uint4 o;
  o.x = pack_bf16x2(q4_value(v, 0, s), q4_value(v, 1, s));
  o.y = pack_bf16x2(q4_value(v, 2, s), q4_value(v, 3, s));
  o.z = pack_bf16x2(q4_value(v, 4, s), q4_value(v, 5, s));
  o.w = pack_bf16x2(q4_value(v, 6, s), q4_value(v, 7, s));
  reinterpret_cast<uint4*>(out + b * bstride + i * ldo + ((int64_t)which * p.Hkv + h) * p.D)[w] = o;
}

// One warp per (sequence, new token, query head), one cached token at a time.
__global__ void __launch_bounds__(256) kv4_attention_kernel(const Kv4AttnParams p) {
  const Kv4Params& kv = p.kv;
  const int lane = threadIdx.x % 32, words = kv.D / 8;
  const int64_t unit = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (unit >= (int64_t)kv.B * kv.L * p.Hq) return;
  const int h = (int)(unit % p.Hq);
  const int64_t row = unit / p.Hq;
  const int b = (int)(row / kv.L), i = (int)(row % kv.L);
  if (i >= new_tokens(kv, b)) return;
  const int pos = position(kv, b, i), hk = h / (p.Hq / kv.Hkv);   // -1: sees nothing, writes zeros
  float q[8], o[8], m = -INFINITY, l = 0.f;
  const __nv_bfloat16* src = p.q + b * p.q_bstride + i * p.q_ld + (int64_t)h * kv.D + lane * 8;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = lane < words ? __bfloat162float(src[e]) * p.scale_log2 : 0.f;
    o[e] = 0.f;
  }
  const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  for (int j = 0; j <= pos; ++j) {
    if (j < lo && j >= p.sinks) j = lo;
    int page = 0;
    if (lane == 0) page = page_of(kv, b, j);
    page = __shfl_sync(0xffffffffu, page, 0);
    if (page < 0) continue;
    float s = 0.f, vs = 0.f;
    uint32_t vw = 0;
    if (lane < words) {
      const int64_t tk = cache_row(kv, page, 0, hk, j), tv = cache_row(kv, page, 1, hk, j);
      const uint32_t kw = reinterpret_cast<const uint32_t*>(kv.codes + tk * (kv.D / 2))[lane];
      const float ks = __bfloat162float(kv.scales[tk * (kv.D / kKvGroup) + lane / 4]);
      vw = reinterpret_cast<const uint32_t*>(kv.codes + tv * (kv.D / 2))[lane];
      vs = __bfloat162float(kv.scales[tv * (kv.D / kKvGroup) + lane / 4]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(q[e], q4_value(kw, e, ks), s);
    }
    s = warp_sum_t(s);
    const float mn = fmaxf(m, s), f = exp2f(m - mn), e2 = exp2f(s - mn);
    m = mn;
    l = l * f + e2;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * f + e2 * q4_value(vw, e, vs);
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (lane < words) {
    __nv_bfloat16* dst = p.out + b * p.o_bstride + i * p.o_ld + (int64_t)h * kv.D + lane * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] = __float2bfloat16_rn(o[e] * inv);
  }
}

template <typename T>
cudaError_t launch_append_t(const Kv4AppendParams& p, unsigned blocks, cudaStream_t stream) {
  switch (p.kv.D) {
    case 64: kv4_append_kernel<T, 1><<<blocks, 256, 0, stream>>>(p); break;
    case 128: kv4_append_kernel<T, 2><<<blocks, 256, 0, stream>>>(p); break;
    case 256: kv4_append_kernel<T, 4><<<blocks, 256, 0, stream>>>(p); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4AppendParams& p, cudaStream_t stream) {
  const int64_t blocks = ((int64_t)p.kv.B * p.kv.L * (p.Hq + 2 * p.kv.Hkv) + 7) / 8;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  return p.in_f32 ? launch_append_t<float>(p, (unsigned)blocks, stream)
                  : launch_append_t<__nv_bfloat16>(p, (unsigned)blocks, stream);
}

cudaError_t launch_kv4_read(const Kv4Params& p, __nv_bfloat16* out, int64_t ldo, int64_t bstride, cudaStream_t stream) {
  const int64_t blocks = ((int64_t)p.B * p.L * 2 * p.Hkv * (p.D / 8) + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  kv4_read_kernel<<<(unsigned)blocks, 256, 0, stream>>>(p, out, ldo, bstride);
  return cudaGetLastError();
}

size_t kv4_attention_workspace(const Kv4AttnParams&) { return 0; }

cudaError_t launch_kv4_attention(const Kv4AttnParams& p, void*, cudaStream_t stream) {
  const int64_t blocks = ((int64_t)p.kv.B * p.kv.L * p.Hq + 7) / 8;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  kv4_attention_kernel<<<(unsigned)blocks, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace nsa
