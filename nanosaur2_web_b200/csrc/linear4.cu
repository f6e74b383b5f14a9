// Linears with 4-bit weights and group scales for a few rows (decode steps): Y = X W^T with
// W[n][k] = s[n][k / G] c[n][k] in the format of q4.cuh, the quantiser that makes such a weight from
// an fp32 / bf16 one, and its expansion back to bf16 (exact), the form nsa_linear takes for many rows.
//
// Layout (made once, at load): rows in tiles of 16, K in chunks of 128, zero padded; a tile's chunk is
// 1024 contiguous bytes [16 rows][64], its scales [16 rows][128 / G] bf16.  Of a row's 64 bytes, the word
// at 16 c + 4 i holds the values 32 i + 8 c .. + 7 (nibble order: q4_nibble).
#include <algorithm>

#include "nsa_internal.h"
#include "ptx.cuh"
#include "q4.cuh"

namespace nsa {

namespace {

constexpr int kRowTile = 16, kChunk = 128;

// byte offset of logical word lw (8 values, 0..15) in a row's 64 bytes of a chunk
__device__ __forceinline__ int word_at(int lw) { return 16 * (lw & 3) + 4 * (lw >> 2); }

// Eight values of a row from k on (zeros past K): one or two 16-byte loads where rows are 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ void load8(const float* row, int k, int K, float* x) {
  if (VEC && k + 8 <= K) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(row + k)), b = __ldg(reinterpret_cast<const float4*>(row + k) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = k + e < K ? row[k + e] : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16* row, int k, int K, float* x) {
  if (VEC && k + 8 <= K) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + k));
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = __uint_as_float(u[e] << 16);
      x[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = k + e < K ? __bfloat162float(row[k + e]) : 0.f;
  }
}

// One CTA per tile chunk, one thread per word (8 values of one row); the 4, 8 or 16 neighbouring threads of a group
// share its largest magnitude by shuffles.  Bound by the weight's bytes.
template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(256) quantize4_kernel(const Quant4Params p) {
  const int tile = blockIdx.x / p.Kc, ch = blockIdx.x % p.Kc;
  const int r = threadIdx.x / 16, w = threadIdx.x % 16;
  const int64_t row = (int64_t)tile * kRowTile + r;
  float x[8];
  if (row < p.N) {
    load8<VEC>(static_cast<const T*>(p.w) + row * p.ldw, ch * kChunk + w * 8, p.K, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  }
  float am = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) am = amax2(fabsf(x[e]), am);
#pragma unroll
  for (int o = 1; o < G / 8; o <<= 1) am = amax2(__shfl_xor_sync(0xffffffffu, am, o), am);
  const float s = q4_scale(am);
  const uint32_t out = s > 0.f ? q4_bits<8, q4_nibble, sizeof(T) == 2>(x, x, s, am) : 0x88888888u;
  const int64_t tr = (int64_t)blockIdx.x * kRowTile + r;   // row of the tiled order
  *reinterpret_cast<uint32_t*>(p.codes + tr * 64 + word_at(w)) = out;
  if (w % (G / 8) == 0) p.scales[tr * (kChunk / G) + w / (G / 8)] = __float2bfloat16_rn(s);
}

// The same shape backwards: a thread per word, one 16-byte store where the rows of out are 16-byte aligned.
template <bool VEC>
__global__ void __launch_bounds__(256) expand4_kernel(const Quant4Params p, __nv_bfloat16* __restrict__ out, int64_t ldo) {
  const int tile = blockIdx.x / p.Kc, ch = blockIdx.x % p.Kc;
  const int r = threadIdx.x / 16, w = threadIdx.x % 16;
  const int64_t row = (int64_t)tile * kRowTile + r;
  const int k = ch * kChunk + w * 8;
  if (row >= p.N || k >= p.K) return;
  const int64_t tr = (int64_t)blockIdx.x * kRowTile + r;
  const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(p.codes + tr * 64 + word_at(w)));
  const uint16_t sc = __ldg(reinterpret_cast<const uint16_t*>(p.scales) + tr * (kChunk / p.G) + w * 8 / p.G);
  __nv_bfloat16* dst = out + row * ldo + k;
  if (VEC && k + 8 <= p.K) {
    uint32_t s2;
    asm("mov.b32 %0, {%1, %1};" : "=r"(s2) : "h"(sc));
    uint4 o;   // code * scale, rounded once
    o.x = mul_bf16x2(code_pair<0>(v), s2);
    o.y = mul_bf16x2(code_pair<1>(v), s2);
    o.z = mul_bf16x2(code_pair<2>(v), s2);
    o.w = mul_bf16x2(code_pair<3>(v), s2);
    *reinterpret_cast<uint4*>(dst) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < p.K) dst[e] = __float2bfloat16_rn(q4_value(v, q4_nibble(e), __uint_as_float((uint32_t)sc << 16)));
  }
}

// ------------------------------------------------------------------------------------ the linear
//
// mma.m16n8k16 with the weight as A (16 rows of a tile) and eight rows of X as B: at these row counts the
// kernel is bound by the weight's bytes, and a tcgen05 tile would need them converted in shared memory first
// (4 times the bytes written and read again), while here each lane loads its 16 bytes of a tile's chunk in the
// A fragment's own order and converts them in registers.  Lane (r, c) holds rows r and r + 8, words i = 0..3 of
// piece c: word i of all four c is group i of 32 values, so one product of k = 32 covers exactly one group,
// starts from zero and enters the row's sum with the group's scale in fp32.  Nibble pairs are neighbours
// (q4_nibble), so X's own 16 bytes of values 32 i + 8 c .. + 7 are the B fragments.  A nibble n set into a bf16
// mantissa is 128 + n; minus 136 it is the code, exactly.
//
// One CTA of 16 warps per SM takes TN = 16 / WK tiles at a time, the WK warps of a tile its chunks in turn, each
// with kStages chunks in flight across tile ends, and joins them in shared memory.  The rows of X that the pass
// covers are staged once per CTA, in the fragments' order.

constexpr int kStages = 4;
constexpr int kWarps = 16;
constexpr int kSmemMax = 227 * 1024;

// Scales of a row's chunk: 128 / G bf16 in one load.
template <int G>
struct ChunkScales;
template <>
struct ChunkScales<32> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = i < 2 ? v.x : v.y;
    return __uint_as_float(i % 2 ? u & 0xFFFF0000u : u << 16);
  }
};
template <>
struct ChunkScales<64> {
  uint32_t v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint32_t*>(p)); }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(i ? v & 0xFFFF0000u : v << 16); }
};
template <>
struct ChunkScales<128> {
  uint16_t v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint16_t*>(p)); }
  __device__ __forceinline__ float get(int) const { return __uint_as_float((uint32_t)v << 16); }
};

// NT: tiles of eight rows of X.
template <int G, int NT>
__global__ void __launch_bounds__(kWarps * 32) linear4_kernel(const Linear4Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kOut = 16 * 8 * NT;                              // values of a tile
  float* red = reinterpret_cast<float*>(smem);                   // [kWarps][m][16]
  uint4* xs = reinterpret_cast<uint4*>(smem + kWarps * kOut * 4);   // [Kc][4 words i][rows][4 pieces c]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
  const int wk = warp % p.WK, tn = warp / p.WK, TN = kWarps / p.WK;
  const int m0 = blockIdx.y * p.rows, rows = min(p.rows, p.M - m0);
  const int steps = (p.Kc + p.WK - 1) / p.WK;                     // chunks of a tile per warp
  const int stride = gridDim.x * TN;
  const int tiles = (p.Nt - (int)blockIdx.x * TN + stride - 1) / stride;   // rounds of this CTA (>= 1)

  uint4 qa[kStages], qb[kStages];
  ChunkScales<G> sa[kStages], sb[kStages];
  int f_tile = blockIdx.x * TN + tn, f_ch = wk, f_left = tiles * steps;   // what the next fetch takes
  int f_step = 0;
  const auto fetch = [&](int st) {
    if (f_left-- > 0 && f_tile < p.Nt && f_ch < p.Kc) {
      const int64_t at = (int64_t)f_tile * p.Kc + f_ch;
      const uint4* codes = reinterpret_cast<const uint4*>(p.codes) + at * 64 + r * 4 + c;
      const __nv_bfloat16* scales = p.scales + (at * 16 + r) * (kChunk / G);
      qa[st] = __ldg(codes);
      qb[st] = __ldg(codes + 32);
      sa[st].load(scales);
      sb[st].load(scales + 8 * (kChunk / G));
    }
    f_ch += p.WK;
    if (++f_step == steps) {
      f_step = 0;
      f_ch = wk;
      f_tile += stride;
    }
  };
#pragma unroll
  for (int st = 0; st < kStages; ++st) fetch(st);

  for (int e = threadIdx.x; e < p.Kc * 16 * rows; e += kWarps * 32) {
    const int w = e / rows, m = e % rows;                         // word w of row m: value 8 w
    const int ch = w / 16, i = w % 16 / 4, cc = w % 4;
    xs[((ch * 4 + i) * rows + m) * 4 + cc] =
        w * 8 < p.K ? __ldg(reinterpret_cast<const uint4*>(p.x + (int64_t)(m0 + m) * p.ldx + w * 8)) : make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();

  // columns past the pass's rows repeat its last row; they are not stored
  const uint4* xt[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) xt[t] = xs + min(8 * t + r, rows - 1) * 4 + c;
  float y[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) y[t][j] = 0.f;
  int tile0 = blockIdx.x * TN, step = 0;
  const int total = tiles * steps;
  for (int f = 0; f < total; f += kStages) {
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      if (f + st >= total) break;
      const int ch = wk + step * p.WK;
      if (ch < p.Kc && tile0 + tn < p.Nt) {
        const uint32_t wa[4] = {qa[st].x, qa[st].y, qa[st].z, qa[st].w}, wb[4] = {qb[st].x, qb[st].y, qb[st].z, qb[st].w};
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (32 * i % G == 0) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[t][j] = 0.f;
          }
          const uint32_t a0 = code_pair<0>(wa[i]), a1 = code_pair<0>(wb[i]), a2 = code_pair<1>(wa[i]), a3 = code_pair<1>(wb[i]);
          const uint32_t a4 = code_pair<2>(wa[i]), a5 = code_pair<2>(wb[i]), a6 = code_pair<3>(wa[i]), a7 = code_pair<3>(wb[i]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint4 x = xt[t][(ch * 4 + i) * rows * 4];
            mma_bf16(acc[t], a0, a1, a2, a3, x.x, x.y);
            mma_bf16(acc[t], a4, a5, a6, a7, x.z, x.w);
          }
          if (32 * (i + 1) % G == 0) {
            const float fa = sa[st].get(32 * i / G), fb = sb[st].get(32 * i / G);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              y[t][0] = fmaf(fa, acc[t][0], y[t][0]);
              y[t][1] = fmaf(fa, acc[t][1], y[t][1]);
              y[t][2] = fmaf(fb, acc[t][2], y[t][2]);
              y[t][3] = fmaf(fb, acc[t][3], y[t][3]);
            }
          }
        }
      }
      fetch(st);
      if (++step < steps) continue;
      // the round's tiles are done: join their warps
      step = 0;
      __syncthreads();   // the previous round's sums have been read
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float* d = red + warp * kOut + (8 * t + 2 * c) * 16 + r;
        d[0] = y[t][0];
        d[16] = y[t][1];
        d[8] = y[t][2];
        d[24] = y[t][3];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[t][j] = 0.f;
      }
      __syncthreads();
      for (int e = threadIdx.x; e < TN * 16 * rows; e += kWarps * 32) {
        const int g = e / (16 * rows), at = e % (16 * rows);
        const int m = m0 + at / 16, n = (tile0 + g) * 16 + at % 16;
        if (n >= p.N) continue;
        float v = 0.f;
        for (int w = 0; w < p.WK; ++w) v += red[(g * p.WK + w) * kOut + at];
        if (p.bias) v += p.bias[n];
        const int64_t o = m * p.ldc + n;
        if (p.out_bf16) static_cast<__nv_bfloat16*>(p.c)[o] = __float2bfloat16_rn(v);
        else if (p.resid) static_cast<float*>(p.c)[o] += v;
        else static_cast<float*>(p.c)[o] = v;
      }
      tile0 += stride;
    }
  }
}

template <int G, int NT>
cudaError_t launch_linear_gn(const Linear4Params& p, dim3 grid, size_t bytes, cudaStream_t stream) {
  static DeviceOnce once;
  const cudaError_t e = once_per_device(once, [] {
    return cudaFuncSetAttribute(linear4_kernel<G, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
  });
  if (e != cudaSuccess) return e;
  linear4_kernel<G, NT><<<grid, kWarps * 32, bytes, stream>>>(p);
  return cudaGetLastError();
}

template <int G>
cudaError_t launch_linear_g(const Linear4Params& p, dim3 grid, cudaStream_t stream) {
  const int nt = (p.rows + 7) / 8;
  const size_t bytes = (size_t)kWarps * 16 * 8 * nt * 4 + (size_t)p.rows * p.Kc * kChunk * 2;
  switch (nt) {
    case 1: return launch_linear_gn<G, 1>(p, grid, bytes, stream);
    case 2: return launch_linear_gn<G, 2>(p, grid, bytes, stream);
    case 3: return launch_linear_gn<G, 3>(p, grid, bytes, stream);
    default: return launch_linear_gn<G, 4>(p, grid, bytes, stream);
  }
}

template <typename T, bool VEC>
cudaError_t launch_quantize_t(const Quant4Params& p, unsigned blocks, cudaStream_t stream) {
  switch (p.G) {
    case 32: quantize4_kernel<T, 32, VEC><<<blocks, 256, 0, stream>>>(p); break;
    case 64: quantize4_kernel<T, 64, VEC><<<blocks, 256, 0, stream>>>(p); break;
    default: quantize4_kernel<T, 128, VEC><<<blocks, 256, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize4(const Quant4Params& p, cudaStream_t stream) {
  const int64_t blocks = (int64_t)p.Nt * p.Kc;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  const bool vec = (reinterpret_cast<uintptr_t>(p.w) | (uintptr_t)(p.ldw * (p.in_f32 ? 4 : 2))) % 16 == 0;
  const unsigned n = (unsigned)blocks;
  if (p.in_f32) return vec ? launch_quantize_t<float, true>(p, n, stream) : launch_quantize_t<float, false>(p, n, stream);
  return vec ? launch_quantize_t<__nv_bfloat16, true>(p, n, stream) : launch_quantize_t<__nv_bfloat16, false>(p, n, stream);
}

cudaError_t launch_expand4(const Quant4Params& p, __nv_bfloat16* out, int64_t ldo, cudaStream_t stream) {
  const int64_t blocks = (int64_t)p.Nt * p.Kc;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ldo * 2)) % 16 == 0)
    expand4_kernel<true><<<(unsigned)blocks, 256, 0, stream>>>(p, out, ldo);
  else
    expand4_kernel<false><<<(unsigned)blocks, 256, 0, stream>>>(p, out, ldo);
  return cudaGetLastError();
}

// Rows of X per pass: up to 32, as many as shared memory holds beside the joins, evenly over the passes.
// Warps per tile: the number with the fewest steps of a warp (rounds of tiles times chunks per warp); of equal
// ones the largest, whose joins are the fewest tiles at a time.
cudaError_t launch_linear4(Linear4Params p, cudaStream_t stream) {
  if (p.Kc > kLinear4MaxK / kChunk) return cudaErrorInvalidValue;
  const int sms = device_sm_count();
  int rows = 32;
  while (rows > 1 && (size_t)kWarps * 16 * 4 * ((rows + 7) / 8 * 8) + (size_t)rows * p.Kc * kChunk * 2 > kSmemMax) --rows;
  const int passes = (p.M + rows - 1) / rows;
  if (passes > 65535) return cudaErrorInvalidValue;
  p.rows = (p.M + passes - 1) / passes;
  int64_t best = INT64_MAX;
  for (int wk = kWarps; wk >= 1; wk /= 2) {
    const int64_t tn = kWarps / wk;
    const int64_t steps = (p.Nt + tn * sms - 1) / (tn * sms) * ((p.Kc + wk - 1) / wk);
    if (steps < best) best = steps, p.WK = wk;
  }
  const int tn = kWarps / p.WK;
  const dim3 grid((unsigned)std::min((p.Nt + tn - 1) / tn, sms), (unsigned)passes);
  switch (p.G) {
    case 32: return launch_linear_g<32>(p, grid, stream);
    case 64: return launch_linear_g<64>(p, grid, stream);
    default: return launch_linear_g<128>(p, grid, stream);
  }
}

}  // namespace nsa
