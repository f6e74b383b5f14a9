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

// One warp per weight row, four rows of X at a time.
__global__ void __launch_bounds__(256) linear4_kernel(const Linear4Params p) {
  const int lane = threadIdx.x % 32;
  const int64_t n = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (n >= p.N) return;
  const int words = p.K / 8, per = kChunk / p.G;
  for (int m0 = 0; m0 < p.M; m0 += 4) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int w = lane; w < words; w += 32) {
      const int64_t tr = ((n / kRowTile) * p.Kc + w / 16) * kRowTile + n % kRowTile;
      const uint32_t v = *reinterpret_cast<const uint32_t*>(p.codes + tr * 64 + word_at(w % 16));
      const float s = __bfloat162float(p.scales[tr * per + (w % 16) * 8 / p.G]);
      for (int m = 0; m < 4 && m0 + m < p.M; ++m) {
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          t = fmaf(q4_value(v, q4_nibble(e), 1.f), __bfloat162float(p.x[(int64_t)(m0 + m) * p.ldx + w * 8 + e]), t);
        acc[m] = fmaf(s, t, acc[m]);
      }
    }
    for (int m = 0; m < 4 && m0 + m < p.M; ++m) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
      if (lane == 0) {
        const float r = acc[m] + (p.bias ? p.bias[n] : 0.f);
        const int64_t at = (int64_t)(m0 + m) * p.ldc + n;
        if (p.out_bf16) static_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(r);
        else if (p.resid) static_cast<float*>(p.c)[at] += r;
        else static_cast<float*>(p.c)[at] = r;
      }
    }
  }
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

cudaError_t launch_linear4(const Linear4Params& p, cudaStream_t stream) {
  linear4_kernel<<<(unsigned)((p.N + 7) / 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace nsa
