// Linears with 4-bit weights and group scales for a few rows (decode steps): Y = X W^T with
// W[n][k] = s[n][k / G] c[n][k] in the format of q4.cuh, the quantiser that makes such a weight from
// an fp32 / bf16 one, and its expansion back to bf16 (exact), the form nsa_linear takes for many rows.
//
// Layout (made once, at load): rows in tiles of 16, K in chunks of 128, zero padded; a tile's chunk is
// 1024 contiguous bytes [16 rows][64], its scales [16 rows][128 / G] bf16.  Of a row's 64 bytes, the word
// at 16 c + 4 i holds the values 32 i + 8 c .. + 7 (nibble order: q4_nibble).
#include <algorithm>

#include <cooperative_groups.h>

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
// share its largest magnitude by shuffles.  8192 x 8200 in groups of 64 takes 55.1 us (5.5 TB/s) from fp32, where the bytes
// bound it, and 61.5 us (2.8 TB/s) from bf16: there 24 warp instructions per 32 values, two roundings each, take 75% of the
// issue slots, and one load a thread leaves 5.6 of 17 cycles per instruction waiting for it.
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

// The same shape backwards: a thread per word, one 16-byte store where the rows of out are 16-byte aligned.  8192 x 8200:
// 43.4 us (3.9 TB/s).  One load and one store a thread in short CTAs: 71% of the issue slots, and half of the cycles between
// a warp's instructions waiting for loads (8.7 of 17); more words a thread would be the next step.
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
// mma.m16n8k16 with the weight as A (16 rows of a tile) and eight rows of X as B: at these row counts the bytes of the
// weight are the floor, and a tcgen05 tile would need them converted in shared memory first
// (4 times the bytes written and read again), while here each lane loads its 16 bytes of a tile's chunk in the
// A fragment's own order and converts them in registers.  Lane (r, c) holds rows r and r + 8, words i = 0..3 of
// piece c: word i of all four c is group i of 32 values, so one product of k = 32 covers exactly one group,
// starts from zero and enters the row's sum with the group's scale in fp32.  Nibble pairs are neighbours
// (q4_nibble), so X's own 16 bytes of values 32 i + 8 c .. + 7 are the B fragments.  A nibble n set into the mantissa
// of 1 / 8 is (1 + n / 128) / 8; minus 17 / 128 it is the code / 1024, exactly, and 128 of them times the largest bf16 do
// not overflow before the scale is applied.
//
// One CTA of 16 warps per SM takes TN = 16 / WK tiles at a time, the WK warps of a tile its chunks in turn.  Each warp
// copies its chunks into a ring of its own, several ahead of their use and across tile ends; the rows of X that the
// pass covers are staged once per CTA, in the fragments' order.  With more rows, staging all of K in every CTA would
// cost more than the weights, so a cluster of CS CTAs shares K: each stages its part of X, goes over the cluster's
// tiles with it, and the parts of the sums are joined through the shared memories at the end.
//
// One row of 16384 x 8192 (group 128) takes 19.4 us (3.6 TB/s; the floor is 10.7); with the products left out the same
// copies take 14.9 us.  (The alternatives below and in linear4_plan were timed beside a form that took 19.0.)
// The rest is instructions: a chunk is 96 of them to convert and 8 products, each of which holds its scheduler for about 5
// cycles.  24 rows of 8200 x 4096 take 15.4 us, 9.4 without the products.  A call of a few hundred kilobytes is its launch
// and one trip to memory: 640 x 1024 in 3.1 us.  Two CTAs per SM with half the registers: 20.7 us instead of 19.0 at
// 16384 x 8192, 6.0 instead of 5.1 at 4096 x 4096.

constexpr int kWarps = 16;
constexpr float kCodeUnit = 1024.f;
constexpr int kSmemMax = 227 * 1024;
constexpr int kMaxCluster = 8;

constexpr int kStages = 3;   // of kStep chunks each; four of them, or six of one chunk, are level or slower (19.0, 20.6 us)
constexpr int kStep = 2;
__host__ __device__ constexpr int stage_bytes(int G) { return kStep * kRowTile * (kChunk / 2 + kChunk / G * 2); }

// Scales of a row's chunk in shared memory: 128 / G bf16 in one load.
template <int G>
struct ChunkScales;
template <>
struct ChunkScales<32> {
  uint2 v;
  __device__ __forceinline__ void load(const uint8_t* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = i < 2 ? v.x : v.y;
    return __uint_as_float(i % 2 ? u & 0xFFFF0000u : u << 16);
  }
};
template <>
struct ChunkScales<64> {
  uint32_t v;
  __device__ __forceinline__ void load(const uint8_t* p) { v = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(i ? v & 0xFFFF0000u : v << 16); }
};
template <>
struct ChunkScales<128> {
  uint32_t v;
  __device__ __forceinline__ void load(const uint8_t* p) { v = *reinterpret_cast<const uint16_t*>(p); }
  __device__ __forceinline__ float get(int) const { return __uint_as_float(v << 16); }
};

__device__ __forceinline__ void write_out(const Linear4Params& p, int m, int n, float v) {
  if (p.bias) v += p.bias[n];
  const int64_t o = m * p.ldc + n;
  if (p.out_bf16) static_cast<__nv_bfloat16*>(p.c)[o] = __float2bfloat16_rn(v);
  else if (p.resid) static_cast<float*>(p.c)[o] += v;
  else static_cast<float*>(p.c)[o] = v;
}

// Codes / kCodeUnit of nibbles P and P + 4 of a word as a bf16 pair.
template <int P>
__device__ __forceinline__ uint32_t small_pair(uint32_t w) {
  uint32_t d;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(mask_or(w >> (4 * P), 0x000F000Fu, 0x3E003E00u)), "r"(0xBE08BE08u));
  return d;
}

// NT: tiles of eight rows of X.
template <int G, int NT>
__global__ void __launch_bounds__(kWarps * 32, 1) linear4_kernel(const Linear4Params p) {
  constexpr int STAGES = kStages, STAGE = stage_bytes(G), CODES = kRowTile * kChunk / 2, SCALES = STAGE / kStep - CODES;   // bytes
  constexpr int kOut = 16 * 8 * NT;                                 // values of a tile
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* rings = smem;                                            // [kWarps][STAGES][STAGE]
  float* red = reinterpret_cast<float*>(smem + kWarps * STAGES * STAGE);   // [kWarps][m][16]
  uint4* xs = reinterpret_cast<uint4*>(red + kWarps * kOut);        // [chunks][4 words i][rows][4 pieces c]
  const int lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int wk = warp % p.WK, tn = warp / p.WK, TN = kWarps / p.WK;
  const int m0 = blockIdx.y * p.rows, rows = min(p.rows, p.M - m0);
  // this CTA's part of K and its cluster's tiles
  const int rank = blockIdx.x % p.CS, each = (p.Kc + p.CS - 1) / p.CS;
  const int c0 = min(rank * each, p.Kc), chunks = min(each, p.Kc - c0);
  const int steps = (each + kStep * p.WK - 1) / (kStep * p.WK);     // of kStep neighbouring chunks of a tile per warp
  const int first = blockIdx.x / p.CS * TN, stride = gridDim.x / p.CS * TN;
  const int rounds = (p.Nt - first + stride - 1) / stride;          // tiles of this cluster, TN at a time (>= 1)
  float* part = reinterpret_cast<float*>(xs + (size_t)each * 16 * p.rows);   // [rounds * TN][rows][16], with CS > 1

  // rows of X: some warps a row, or some rows a warp, 16 bytes a lane (zeros past K)
  {
    int share = 1;                                                  // warps per row
    while (2 * share * rows <= kWarps) share *= 2;
    const uint32_t to = smem_u32(xs);
    for (int m = warp / share; m < rows; m += kWarps / share) {
      const __nv_bfloat16* src = p.x + (int64_t)(m0 + m) * p.ldx;
      for (int w = (warp % share) * 32 + lane; w < chunks * 16; w += share * 32) {
        const int k = c0 * kChunk + w * 8;
        copy16_async_fill(to + (((w / 4) * rows + m) * 4 + w % 4) * 16, src + (k < p.K ? k : 0), k < p.K ? 16 : 0);
      }
    }
    copy_commit();
  }

  const uint32_t ring = smem_u32(rings) + warp * STAGES * STAGE;
  // a stage: kStep chunks' codes, then their scales
  const uint8_t* codes = p.codes + lane * 16;
  const uint8_t* scales = reinterpret_cast<const uint8_t*>(p.scales) + lane * 16;
  int f_tile = first + tn, f_step = 0, f_stage = 0;                 // what the next fetch takes, and where
  const auto fetch = [&] {
    const int ch = (f_step * p.WK + wk) * kStep;
    if (f_tile < p.Nt && ch < chunks) {
      const uint64_t at = (uint32_t)f_tile * (uint32_t)p.Kc + (uint32_t)(c0 + ch);
      const uint32_t to = ring + f_stage * STAGE + lane * 16;
      const uint8_t* src = codes + at * CODES;
      copy16_async(to, src);
      copy16_async(to + 512, src + 512);
      if (ch + 1 < chunks) {
        copy16_async(to + 1024, src + 1024);
        copy16_async(to + 1536, src + 1536);
      }
      if (lane * 16 < (ch + 1 < chunks ? 2 : 1) * SCALES) copy16_async(to + kStep * CODES, scales + at * SCALES);
    }
    copy_commit();
    f_stage = f_stage == STAGES - 1 ? 0 : f_stage + 1;
    if (++f_step == steps) {
      f_step = 0;
      f_tile += stride;
    }
  };
#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st) fetch();
  copy_wait<STAGES - 1>();   // X
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
  int stage = 0;
  for (int round = 0; round < rounds; ++round) {
    const int tile0 = first + round * stride;
    for (int step = 0; step < steps; ++step) {
      copy_wait<STAGES - 2>();
      __syncwarp();   // the chunks are there for all lanes, and all lanes are done with the stage that is filled next
      fetch();
      const uint8_t* at = rings + (warp * STAGES + stage) * STAGE;
      stage = stage == STAGES - 1 ? 0 : stage + 1;
      const int ch = (step * p.WK + wk) * kStep;
      if (ch >= chunks || tile0 + tn >= p.Nt) continue;
      const auto multiply = [&](int half) {
        const uint4 qa = *reinterpret_cast<const uint4*>(at + half * CODES + r * 64 + c * 16);
        const uint4 qb = *reinterpret_cast<const uint4*>(at + half * CODES + (r + 8) * 64 + c * 16);
        ChunkScales<G> sa, sb;
        sa.load(at + kStep * CODES + half * SCALES + r * (kChunk / G * 2));
        sb.load(at + kStep * CODES + half * SCALES + (r + 8) * (kChunk / G * 2));
        const uint32_t wa[4] = {qa.x, qa.y, qa.z, qa.w}, wb[4] = {qb.x, qb.y, qb.z, qb.w};
        const int xo = (ch + half) * 16 * rows;
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = small_pair<0>(wa[i]), a1 = small_pair<0>(wb[i]), a2 = small_pair<1>(wa[i]), a3 = small_pair<1>(wb[i]);
          const uint32_t a4 = small_pair<2>(wa[i]), a5 = small_pair<2>(wb[i]), a6 = small_pair<3>(wa[i]), a7 = small_pair<3>(wb[i]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint4 x = xt[t][xo + i * 4 * rows];
            if (32 * i % G == 0) mma_bf16_zero(acc[t], a0, a1, a2, a3, x.x, x.y);
            else mma_bf16(acc[t], a0, a1, a2, a3, x.x, x.y);
            mma_bf16(acc[t], a4, a5, a6, a7, x.z, x.w);
          }
          if (32 * (i + 1) % G == 0) {
            const float fa = sa.get(32 * i / G), fb = sb.get(32 * i / G);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              y[t][0] = fmaf(fa, acc[t][0], y[t][0]);
              y[t][1] = fmaf(fa, acc[t][1], y[t][1]);
              y[t][2] = fmaf(fb, acc[t][2], y[t][2]);
              y[t][3] = fmaf(fb, acc[t][3], y[t][3]);
            }
          }
        }
      };
      multiply(0);
      if (ch + 1 < chunks) multiply(1);
    }
    // the round's tiles are done: join their warps
    __syncthreads();   // the previous round's sums have been read
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float* d = red + warp * kOut + (8 * t + 2 * c) * 16 + r;
      d[0] = y[t][0] * kCodeUnit;
      d[16] = y[t][1] * kCodeUnit;
      d[8] = y[t][2] * kCodeUnit;
      d[24] = y[t][3] * kCodeUnit;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[t][j] = 0.f;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < TN * kOut; e += kWarps * 32) {
      const int g = e / kOut, at = e % kOut, m = at / 16, n = (tile0 + g) * 16 + at % 16;
      if (m >= rows) continue;
      float v = 0.f;
      for (int w = 0; w < p.WK; ++w) v += red[(g * p.WK + w) * kOut + at];
      if (p.CS > 1) part[((round * TN + g) * rows + m) * 16 + at % 16] = v;
      else if (n < p.N) write_out(p, m0 + m, n, v);
    }
  }
  if (p.CS > 1) {
    const auto cluster = cooperative_groups::this_cluster();
    cluster.sync();
    for (int e = rank * kWarps * 32 + threadIdx.x; e < rounds * TN * rows * 16; e += p.CS * kWarps * 32) {
      const int j = e / 16 / rows, m = e / 16 - j * rows, n = (first + j / TN * stride + j % TN) * 16 + e % 16;
      if (n >= p.N) continue;
      float v = 0.f;
      for (int k = 0; k < p.CS; ++k) v += *cluster.map_shared_rank(part + e, k);
      write_out(p, m0 + m, n, v);
    }
    cluster.sync();   // no CTA leaves while another reads its shared memory
  }
}

template <int G, int NT>
cudaError_t launch_linear_gn(const Linear4Params& p, dim3 grid, size_t bytes, cudaStream_t stream) {
  static DeviceOnce once;
  const cudaError_t e = once_per_device(once, [] {
    return cudaFuncSetAttribute(linear4_kernel<G, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = p.CS;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = p.CS > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, linear4_kernel<G, NT>, p);
}

template <int G>
cudaError_t launch_linear_g(const Linear4Params& p, dim3 grid, size_t bytes, cudaStream_t stream) {
  switch ((p.rows + 7) / 8) {
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

namespace {

// A way to share the work of a pass of `rows` rows, and its estimated cycles.  What it decides, measured in us:
//   warps per tile    16384 x 8192, 1 row: 2 take 19.0, 16 19.1, 4 19.4;  4096 x 4096: 8 take 5.1, 16 5.5, 4 7.1, 2 8.2
//   CTAs that share K  16384 x 8192, 1 row: 1 takes 19.0, 2 19.7, 4 23.2;  24 rows of 8200 x 4096 fit only from 4 on
struct Linear4Plan {
  int WK, CS, clusters;
  size_t bytes;
  double cost;
};

Linear4Plan linear4_plan(const Linear4Params& p, int rows, int sms) {
  const int nt = (rows + 7) / 8;
  Linear4Plan best{0, 0, 0, 0, 1e30};
  for (int cs = 1; cs <= kMaxCluster; cs *= 2) {
    if (cs > 1 && cs > p.Kc) break;
    // clusters of 8 or 4 CTAs leave a few SMs of a processing cluster over
    const int clusters = cs == 1 ? sms : cs == 2 ? sms / 2 : cs == 4 ? sms / 4 - 1 : sms / 8 - 2;
    const int64_t each = (p.Kc + cs - 1) / cs;
    for (int wk = kWarps; wk >= 1; wk /= 2) {
      const int64_t tn = kWarps / wk, rounds = (p.Nt + tn * clusters - 1) / (tn * clusters);
      const size_t bytes = (size_t)kWarps * kStages * stage_bytes(p.G) + (size_t)kWarps * 16 * 8 * nt * 4 +
                           (size_t)each * 256 * rows + (cs > 1 ? (size_t)rounds * tn * rows * 64 : 0);
      if (bytes > kSmemMax) continue;
      // a step: the instructions of a scheduler's warps; a round: its join; X at about 48 bytes a cycle; a
      // cluster's join
      const double cost = (double)rounds * ((each + kStep * wk - 1) / (kStep * wk)) * kStep * 4 * (150 + 50 * nt) * 1.6 +
                          rounds * 800.0 + each * 256.0 * rows / 48 + (cs > 1 ? 1500.0 : 0.0);
      if (cost < best.cost) best = {wk, cs, (int)std::min<int64_t>(clusters, (p.Nt + tn - 1) / tn), bytes, cost};
    }
  }
  return best;
}

}  // namespace

// Rows of X per pass: up to 32, fewer where no cluster holds them, evenly over the passes; passes are the grid's second
// axis, of at most 65535.  cudaErrorNotSupported: not even one row fits.
cudaError_t launch_linear4(Linear4Params p, cudaStream_t stream) {
  const int sms = device_sm_count();
  int most = std::min(p.M, 32);
  Linear4Plan plan = linear4_plan(p, most, sms);
  while (plan.WK == 0 && most > 1) plan = linear4_plan(p, --most, sms);
  if (plan.WK == 0) return cudaErrorNotSupported;
  const int size = p.out_bf16 ? 2 : 4;
  for (int left = p.M; left > 0; left -= p.M) {
    p.M = (int)std::min<int64_t>(left, (int64_t)most * 65535);
    const int passes = (p.M + most - 1) / most;
    p.rows = (p.M + passes - 1) / passes;
    plan = linear4_plan(p, p.rows, sms);
    p.WK = plan.WK;
    p.CS = plan.CS;
    const dim3 grid((unsigned)(plan.clusters * p.CS), (unsigned)passes);
    const cudaError_t e = p.G == 32   ? launch_linear_g<32>(p, grid, plan.bytes, stream)
                          : p.G == 64 ? launch_linear_g<64>(p, grid, plan.bytes, stream)
                                      : launch_linear_g<128>(p, grid, plan.bytes, stream);
    if (e != cudaSuccess) return e;
    p.x += (int64_t)p.M * p.ldx;
    p.c = static_cast<char*>(p.c) + (int64_t)p.M * p.ldc * size;
  }
  return cudaSuccess;
}

}  // namespace nsa
