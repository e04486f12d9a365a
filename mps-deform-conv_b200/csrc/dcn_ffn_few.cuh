// dcn_ffn_few.cuh -- the gated feed-forward block on few rows (single vectors and
// small batches while serving), forward only.
//
// What bounds it: the weights, 3 C F values read once for at most 32 rows; at
// one row every weight takes part in one multiplication.  Two kernels, each
// streaming its weights from HBM straight into registers:
//   few_gate_up   hidden[m][f] = act(x Wg^T + bg) * (x Wu^T + bu)
//   few_down      y[m][c] = hidden Wd^T + bd
// A warp takes 16 weight rows (of gate and of up, or of down) and K in blocks of
// 64; a lane reads 16-byte pieces, four lanes a 64-byte run of a row.  The four
// warps of a CTA take different rows (they read the same part of x, which then
// comes from the L1), or with few weight rows the same ones and share K; a
// cluster of up to eight CTAs shares K too, so that a product with few weight
// rows still keeps every SM loading.  16-bit data multiplies with the
// legacy warp-level matrix instruction (rows of weights as the 16 x 16 operand,
// up to 8 rows of x as the other): it takes its operands from registers, and at
// this intensity (2 flops a byte and row) its rate does not matter.  The order
// of a contraction is free, so a lane's eight consecutive values serve as its
// share of two instructions' operands, x read the same way.  fp32 data
// multiplies on the CUDA cores.  The warps' sums meet in shared memory, the
// CTAs' in each other's, both in a fixed order.  The hidden values are rounded to
// the data's type between the two kernels, where the tile products round them too.
//
// Measured (back-to-back calls in a graph): one row through 512 -> 2048 in bf16
// 6.9 us, of it 1 us of weights at the memory's rate: two launches and their
// first loads; through 4096 -> 14336 68 us, 5.2 TB/s of weights.
//
// few_down starts while few_gate_up runs (programmatic launch): it fetches its
// first weights and waits for the hidden values only then.
#pragma once

#include <type_traits>

#include "dcn_ffn_gemm.cuh"

namespace dcn {
namespace ffn {

constexpr int kFewRows = 32;     // most rows of x
constexpr int kFewTile = 16;     // weight rows of a warp

struct FewArgs {
  const void* x;       // [M][K]
  const void* w[2];    // [N][K]: gate and up, or down
  const void* bias[2];
  void* out;           // [M][N]
  int M, N, K, act;
};

__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Weights are read once: past the L1.
__device__ __forceinline__ uint4 load_weights(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float load_cluster(const float* p, uint32_t rank) {
  uint32_t addr;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// 16-bit data.  NT: groups of 8 rows of x; GATED: gate and up, else plain; ROWS:
// the warps take different weight rows, else they share K.  The CTAs of a
// cluster share a tile.  K a multiple of 8, all rows on 16-byte boundaries.
constexpr int kFewWarps = 4;
template <typename T, bool GATED, int NT, bool ROWS>
__global__ void __launch_bounds__(kFewWarps * 32) ffn_few_kernel(const __grid_constant__ FewArgs a, int ctas) {
  constexpr int SETS = GATED ? 2 : 1, WARPS = kFewWarps;
  constexpr int TILE = kFewTile * (ROWS ? WARPS : 1), KW = ROWS ? 1 : WARPS;  // weight rows of a tile; warps that share K
  __shared__ float sums[KW][SETS][TILE][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = ctas > 1 ? (int)cluster_rank() : 0;
  const int tile0 = (blockIdx.x / ctas) * TILE, n0 = tile0 + (ROWS ? warp * kFewTile : 0);
  const T* w[SETS][2];  // this lane's two weight rows; rows past N read row N - 1, their sums are not stored
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[s][i] = static_cast<const T*>(a.w[s]) + (int64_t)min(n0 + g + 8 * i, a.N - 1) * a.K + t * 8;
  const T* x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = static_cast<const T*>(a.x) + (int64_t)min(8 * n + g, a.M - 1) * a.K + t * 8;

  float acc[SETS][NT][4];
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[s][n][j] = 0.0f;

  const int blocks = (a.K + 63) / 64, step = KW * ctas;
  uint4 r[SETS][2][2];  // [set][row][piece]
  auto fetch = [&](int b) {
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int k = b * 64 + p * 32;
          r[s][i][p] = k + t * 8 < a.K ? load_weights(w[s][i] + k) : make_uint4(0, 0, 0, 0);
        }
  };
  int b = rank * KW + (ROWS ? 0 : warp);
  if (b < blocks) fetch(b);
  if (GATED) pdl_launch();
  else pdl_wait();  // x is the previous kernel's result
#pragma unroll 2
  for (; b < blocks; b += step) {
    uint4 v[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int k = b * 64 + p * 32;
        v[n][p] = k + t * 8 < a.K ? *reinterpret_cast<const uint4*>(x[n] + k) : make_uint4(0, 0, 0, 0);
      }
    uint4 c[SETS][2][2];
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) c[s][i][p] = r[s][i][p];
    if (b + step < blocks) fetch(b + step);
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          const uint4 &r0 = c[s][0][p], &r1 = c[s][1][p], &q = v[n][p];
          mma_16816<T>(acc[s][n], r0.x, r1.x, r0.y, r1.y, q.x, q.y);
          mma_16816<T>(acc[s][n], r0.z, r1.z, r0.w, r1.w, q.z, q.w);
        }
  }
  // lane (g, t): weight rows g, g + 8; rows 2 t, 2 t + 1 of each group of x
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[ROWS ? 0 : warp][s][n0 - tile0 + g + 8 * (j >> 1)][8 * n + 2 * t + (j & 1)] = acc[s][n][j];
  __syncthreads();
  auto finish = [&](int i, auto&& sum) {
    const int row = i % TILE, m = i / TILE, c = tile0 + row;  // consecutive lanes: consecutive outputs of a row
    if (c >= a.N || m >= a.M) return;
    float v[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      v[s] = sum(s, row, m);
      if (a.bias[s]) v[s] += to_f<T>(static_cast<const T*>(a.bias[s])[c]);
    }
    float o = v[0];
    if constexpr (GATED) {
      o = (a.act == kActSilu   ? act_value<false, kActSilu>(v[0])
           : a.act == kActGelu ? act_value<false, kActGelu>(v[0])
           : a.act == kActRelu ? act_value<false, kActRelu>(v[0])
                               : act_value<false, kActSigmoid>(v[0])) * v[1];
    }
    static_cast<T*>(a.out)[(int64_t)m * a.N + c] = from_f<T>(o);
  };
  if (ctas == 1) {
    for (int i = threadIdx.x; i < TILE * 8 * NT; i += WARPS * 32)
      finish(i, [&](int s, int row, int m) {
        float v = sums[0][s][row][m];
#pragma unroll
        for (int q = 1; q < KW; ++q) v += sums[q][s][row][m];
        return v;
      });
    return;
  }
  if (KW > 1) {  // this CTA's part, over its warps
    for (int i = threadIdx.x; i < TILE * 8 * NT; i += WARPS * 32)
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        float v = sums[0][s][i % TILE][i / TILE];
#pragma unroll
        for (int q = 1; q < KW; ++q) v += sums[q][s][i % TILE][i / TILE];
        sums[0][s][i % TILE][i / TILE] = v;
      }
  }
  cluster_sync();
  // each CTA finishes its share of the tile from all parts, in order
  for (int i = rank * WARPS * 32 + threadIdx.x; i < TILE * 8 * NT; i += ctas * WARPS * 32)
    finish(i, [&](int s, int row, int m) {
      float v = 0.0f;
      for (int q = 0; q < ctas; ++q) v += load_cluster(&sums[0][s][row][m], (uint32_t)q);
      return v;
    });
  cluster_sync();  // the parts are read
}

// fp32 data: a warp takes one weight row (of gate and of up), lanes share K;
// eight rows of x at a time.  Grid: (weight rows / 8, groups of 8 rows of x).
template <bool GATED>
__global__ void __launch_bounds__(256) ffn_few_f32_kernel(const __grid_constant__ FewArgs a) {
  constexpr int SETS = GATED ? 2 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x * 8 + warp, m0 = blockIdx.y * 8;
  if (GATED) pdl_launch();
  else pdl_wait();
  if (c >= a.N) return;
  const float* w[SETS];
#pragma unroll
  for (int s = 0; s < SETS; ++s) w[s] = static_cast<const float*>(a.w[s]) + (int64_t)c * a.K;
  const float* x = static_cast<const float*>(a.x) + (int64_t)m0 * a.K;
  const int rows = min(8, a.M - m0);
  float acc[SETS][8];
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int m = 0; m < 8; ++m) acc[s][m] = 0.0f;
  if (a.K % 4 == 0) {
#pragma unroll 2
    for (int k = lane * 4; k < a.K; k += 128) {
      float4 v[SETS];
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        const uint4 r = load_weights(w[s] + k);
        v[s] = make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w));
      }
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        if (m >= rows) break;
        const float4 q = *reinterpret_cast<const float4*>(x + (int64_t)m * a.K + k);
#pragma unroll
        for (int s = 0; s < SETS; ++s)
          acc[s][m] = fmaf(v[s].x, q.x, fmaf(v[s].y, q.y, fmaf(v[s].z, q.z, fmaf(v[s].w, q.w, acc[s][m]))));
      }
    }
  } else {
    for (int k = lane; k < a.K; k += 32) {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        if (m >= rows) break;
        const float q = x[(int64_t)m * a.K + k];
#pragma unroll
        for (int s = 0; s < SETS; ++s) acc[s][m] = fmaf(w[s][k], q, acc[s][m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    if (m >= rows) break;
    float v[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      v[s] = acc[s][m];
#pragma unroll
      for (int o = 16; o; o >>= 1) v[s] += __shfl_xor_sync(0xffffffffu, v[s], o);
      if (a.bias[s]) v[s] += static_cast<const float*>(a.bias[s])[c];
    }
    float o = v[0];
    if constexpr (GATED) {
      o = (a.act == kActSilu   ? act_value<true, kActSilu>(v[0])
           : a.act == kActGelu ? act_value<true, kActGelu>(v[0])
           : a.act == kActRelu ? act_value<true, kActRelu>(v[0])
                               : act_value<true, kActSigmoid>(v[0])) * v[1];
    }
    if (lane == 0) static_cast<float*>(a.out)[(int64_t)(m0 + m) * a.N + c] = o;
  }
}

// `dependent`: may start before the launch in front of it has ended (it waits itself).
template <typename K, typename... Rest>
cudaError_t launch_few(const char* name, K kern, dim3 grid, int threads, int cluster, bool dependent, cudaStream_t st,
                       const FewArgs& a, Rest... rest) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (dependent) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = (unsigned)n;
  KernelScope ks(name, st);
  return cudaLaunchKernelEx(&cfg, kern, a, rest...);
}

template <typename T, bool GATED>
cudaError_t launch_few(const char* name, const FewArgs& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 4) {
    return launch_few(name, ffn_few_f32_kernel<GATED>, dim3((unsigned)div_up(a.N, 8), (unsigned)div_up(a.M, 8)), 256, 1,
                      !GATED, st, a);
  } else {
    // Warps on different rows where that leaves at least four CTAs an SM with K
    // in eight parts.  CTAs of a tile: doubled while all tiles together are fewer
    // than six CTAs an SM and every warp keeps a block of K.
    const int64_t blocks = div_up(a.K, 64);
    const bool rows = div_up(a.N, kFewTile * kFewWarps) * std::min<int64_t>(8, blocks) >= 4 * kSms;
    const int64_t tiles = div_up(a.N, kFewTile * (rows ? kFewWarps : 1));
    int ctas = 1;
    while (ctas < 8 && tiles * ctas < 6 * kSms && 2 * ctas * (rows ? 1 : kFewWarps) <= blocks) ctas *= 2;
    auto go = [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      const dim3 grid((unsigned)(tiles * ctas));
      const int threads = kFewWarps * 32;
      return rows ? launch_few(name, ffn_few_kernel<T, GATED, NT, true>, grid, threads, ctas, !GATED, st, a, ctas)
                  : launch_few(name, ffn_few_kernel<T, GATED, NT, false>, grid, threads, ctas, !GATED, st, a, ctas);
    };
    if (a.M <= 8) return go(std::integral_constant<int, 1>{});
    if (a.M <= 16) return go(std::integral_constant<int, 2>{});
    return go(std::integral_constant<int, 4>{});
  }
}

}  // namespace ffn
}  // namespace dcn
