// Linears with 4-bit weights and group scales for a few rows (decode steps): Y = X W^T with
// W[n][k] = s[n][k / G] c[n][k] in the format of q4.cuh, the quantiser that makes such a weight from
// an fp32 / bf16 one, and its expansion back to bf16 (exact), the form nsa_linear takes for many rows.
//
// Layout (made once, at load): rows in tiles of 16, K in chunks of 128, zero padded; a tile's chunk is
// 1024 contiguous bytes [16 rows][64], its scales [16 rows][128 / G] bf16.  Of a row's 64 bytes, the word
// at 16 c + 4 i holds the values 32 i + 8 c .. + 7 (nibble order: q4_nibble).
#include "nsa_internal.h"
#include "q4.cuh"

namespace nsa {

namespace {

constexpr int kRowTile = 16, kChunk = 128;

// byte offset of logical word lw (8 values, 0..15) in a row's 64 bytes of a chunk
__device__ __forceinline__ int word_at(int lw) { return 16 * (lw & 3) + 4 * (lw >> 2); }

template <typename T>
__device__ __forceinline__ float load1(const void* p, int64_t i);
template <>
__device__ __forceinline__ float load1<float>(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
template <>
__device__ __forceinline__ float load1<__nv_bfloat16>(const void* p, int64_t i) {
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// One thread per word (8 values of one row); the 4, 8 or 16 neighbouring threads of a group share its
// largest magnitude by shuffles.
template <typename T, int G>
__global__ void __launch_bounds__(256) quantize4_kernel(const Quant4Params p) {
  const int64_t words = (int64_t)p.Kc * 16;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;   // grid covers Nt * 16 rows x words exactly
  const int64_t row = idx / words;
  const int w = (int)(idx % words);
  if (row >= (int64_t)p.Nt * kRowTile) return;                   // whole warps: words is a multiple of 16 and rows of 16
  float x[8];
  float am = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = w * 8 + e;
    x[e] = (row < p.N && k < p.K) ? load1<T>(p.w, row * p.ldw + k) : 0.f;
    am = amax2(fabsf(x[e]), am);
  }
#pragma unroll
  for (int o = 1; o < G / 8; o <<= 1) am = amax2(__shfl_xor_sync(0xffffffffu, am, o), am);
  const float s = q4_scale(am);
  uint32_t out = 0x88888888u;
  if (s > 0.f) {
    const float inv = __fdiv_rn(1.f, s);
    out = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) out |= q4_code(x[e], s, inv) << (4 * q4_nibble(e));
  }
  const int64_t tr = ((row / kRowTile) * p.Kc + w / 16) * kRowTile + row % kRowTile;   // row of the tiled order
  *reinterpret_cast<uint32_t*>(p.codes + tr * 64 + word_at(w % 16)) = out;
  if (w % (G / 8) == 0) p.scales[tr * (kChunk / G) + (w % 16) / (G / 8)] = __float2bfloat16_rn(s);
}

__global__ void __launch_bounds__(256) expand4_kernel(const Quant4Params p, __nv_bfloat16* __restrict__ out, int64_t ldo) {
  const int64_t words = (p.K + 7) / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / words;
  const int w = (int)(idx % words);
  if (row >= p.N) return;
  const int64_t tr = ((row / kRowTile) * p.Kc + w / 16) * kRowTile + row % kRowTile;
  const uint32_t v = *reinterpret_cast<const uint32_t*>(p.codes + tr * 64 + word_at(w % 16));
  const int per = kChunk / p.G;
  const float s = __bfloat162float(p.scales[tr * per + (w % 16) * 8 / p.G]);
  for (int e = 0; e < 8 && w * 8 + e < p.K; ++e)
    out[row * ldo + w * 8 + e] = __float2bfloat16_rn(q4_value(v, q4_nibble(e), s));
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
// A tile's chunks are one contiguous stream, shared by WK warps of the CTA (chunk k to warp k % WK) and joined
// in shared memory; each warp keeps kStages chunks in flight.

constexpr int kStages = 4;

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

template <int P>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t d;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(((w >> (4 * P)) & 0x000F000Fu) | 0x43004300u), "r"(0xC308C308u));
  return d;
}

// NT: tiles of eight rows of X.
template <int G, int NT>
__global__ void __launch_bounds__(256) linear4_kernel(const Linear4Params p) {
  __shared__ float red[8][16 * 8 * NT];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
  const int wk = warp % p.WK, tile = blockIdx.x * (8 / p.WK) + warp / p.WK;
  const int m0 = blockIdx.y * 8 * NT;
  float y[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) y[t][j] = 0.f;
  if (tile < p.Nt) {
    const uint4* codes = reinterpret_cast<const uint4*>(p.codes) + ((int64_t)tile * p.Kc * 16 + r) * 4 + c;
    const __nv_bfloat16* scales = p.scales + ((int64_t)tile * p.Kc * 16 + r) * (kChunk / G);
    uint4 qa[kStages], qb[kStages];
    ChunkScales<G> sa[kStages], sb[kStages];
    const auto fetch = [&](int st, int ch) {
      if (ch >= p.Kc) return;
      qa[st] = __ldg(codes + (int64_t)ch * 64);
      qb[st] = __ldg(codes + (int64_t)ch * 64 + 32);
      sa[st].load(scales + (int64_t)ch * (16 * kChunk / G));
      sb[st].load(scales + (int64_t)ch * (16 * kChunk / G) + 8 * (kChunk / G));
    };
#pragma unroll
    for (int st = 0; st < kStages; ++st) fetch(st, wk + st * p.WK);
    for (int base = wk; base < p.Kc; base += kStages * p.WK) {
#pragma unroll
      for (int st = 0; st < kStages; ++st) {
        const int ch = base + st * p.WK;
        if (ch >= p.Kc) break;
        const uint32_t wa[4] = {qa[st].x, qa[st].y, qa[st].z, qa[st].w}, wb[4] = {qb[st].x, qb[st].y, qb[st].z, qb[st].w};
        const ChunkScales<G> ca = sa[st], cb = sb[st];
        fetch(st, ch + kStages * p.WK);
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = ch * kChunk + 32 * i + 8 * c;
          uint4 x[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const int m = m0 + 8 * t + r;
            x[t] = m < p.M && k < p.K ? __ldg(reinterpret_cast<const uint4*>(p.x + m * p.ldx + k)) : make_uint4(0u, 0u, 0u, 0u);
          }
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
            mma_bf16(acc[t], a0, a1, a2, a3, x[t].x, x[t].y);
            mma_bf16(acc[t], a4, a5, a6, a7, x[t].z, x[t].w);
          }
          if (32 * (i + 1) % G == 0) {
            const float fa = ca.get(32 * i / G), fb = cb.get(32 * i / G);
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
    }
  }
  // red[warp][m][n]
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float* d = red[warp] + (8 * t + 2 * c) * 16 + r;
    d[0] = y[t][0];
    d[16] = y[t][1];
    d[8] = y[t][2];
    d[24] = y[t][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < (8 / p.WK) * 16 * 8 * NT; e += 256) {
    const int g = e / (16 * 8 * NT), at = e % (16 * 8 * NT);
    const int m = m0 + at / 16, n = (blockIdx.x * (8 / p.WK) + g) * 16 + at % 16;
    if (m >= p.M || n >= p.N) continue;
    float v = 0.f;
    for (int w = 0; w < p.WK; ++w) v += red[g * p.WK + w][at];
    if (p.bias) v += p.bias[n];
    const int64_t o = m * p.ldc + n;
    if (p.out_bf16) static_cast<__nv_bfloat16*>(p.c)[o] = __float2bfloat16_rn(v);
    else if (p.resid) static_cast<float*>(p.c)[o] += v;
    else static_cast<float*>(p.c)[o] = v;
  }
}

template <int G>
cudaError_t launch_linear_g(const Linear4Params& p, cudaStream_t stream) {
  const int nt = p.M >= 32 ? 4 : (p.M + 7) / 8;
  const dim3 grid((unsigned)((p.Nt + 8 / p.WK - 1) / (8 / p.WK)), (unsigned)((p.M + 8 * nt - 1) / (8 * nt)));
  if (grid.y > 65535) return cudaErrorInvalidValue;
  switch (nt) {
    case 1: linear4_kernel<G, 1><<<grid, 256, 0, stream>>>(p); break;
    case 2: linear4_kernel<G, 2><<<grid, 256, 0, stream>>>(p); break;
    case 3: linear4_kernel<G, 3><<<grid, 256, 0, stream>>>(p); break;
    default: linear4_kernel<G, 4><<<grid, 256, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_quantize_t(const Quant4Params& p, cudaStream_t stream) {
  const int64_t blocks = (int64_t)p.Nt * p.Kc;   // 16 rows x 16 words = 256 threads per tile chunk
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  switch (p.G) {
    case 32: quantize4_kernel<T, 32><<<(unsigned)blocks, 256, 0, stream>>>(p); break;
    case 64: quantize4_kernel<T, 64><<<(unsigned)blocks, 256, 0, stream>>>(p); break;
    default: quantize4_kernel<T, 128><<<(unsigned)blocks, 256, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize4(const Quant4Params& p, cudaStream_t stream) {
  return p.in_f32 ? launch_quantize_t<float>(p, stream) : launch_quantize_t<__nv_bfloat16>(p, stream);
}

cudaError_t launch_expand4(const Quant4Params& p, __nv_bfloat16* out, int64_t ldo, cudaStream_t stream) {
  const int64_t blocks = ((int64_t)p.N * ((p.K + 7) / 8) + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  expand4_kernel<<<(unsigned)blocks, 256, 0, stream>>>(p, out, ldo);
  return cudaGetLastError();
}

// Warps per tile: as few as give every SM 16 warps (a warp's own stream is longer and its join cheaper), but
// no more than a tile has chunks.
cudaError_t launch_linear4(Linear4Params p, cudaStream_t stream) {
  p.WK = 1;
  while (p.WK < 8 && (int64_t)p.Nt * p.WK < 16 * 148 && 2 * p.WK <= p.Kc) p.WK *= 2;
  switch (p.G) {
    case 32: return launch_linear_g<32>(p, stream);
    case 64: return launch_linear_g<64>(p, stream);
    default: return launch_linear_g<128>(p, stream);
  }
}

}  // namespace nsa
