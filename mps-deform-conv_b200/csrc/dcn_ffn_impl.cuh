// dcn_ffn_impl.cuh -- the gated feed-forward block, forward and backward:
//   gate = x Wg^T + bg, up = x Wu^T + bu, hidden = act(gate) * up, y = hidden Wd^T + bd
//   dhidden = dy Wd, dgate = dhidden * up * act'(gate), dup = dhidden * act(gate)
//   dx = dgate Wg + dup Wu, dWg = dgate^T x, dWu = dup^T x, dWd = dy^T hidden, db = column sums
// Every product is ffn_gemm_kernel (dcn_ffn_gemm.cuh); this file plans the
// launches, packs operands that the TMA cannot read in place, and finishes
// sums that were split.  dcn_ffn_{bf16,fp16,fp32}.cu instantiate it.
//
// Work: 6 M C F flops forward, 12 M C F backward (M rows, C channels, F hidden).
// Measured, forward and backward: 92416 x 512 -> 2048 in bf16 1.75 ms of kernels
// (1.0 PFLOP/s; 2.06 to 2.08 ms once steady calls reach the power cap), 921600 x
// 64 -> 170 in fp16 0.88 ms, 8192 x 128 -> 512 in fp32 0.26 ms.
// The hidden values and the two hidden gradients are rounded to the data's
// type, as operands of the following products; everything else stays in 32
// bits to the final rounding.
#pragma once

#include <algorithm>
#include <vector>

#include "dcn_ffn_few.cuh"
#include "dcn_ffn_gemm.cuh"
#include "dcn_ffn_layout.h"

namespace dcn {

using namespace ffn;

namespace {

// ---------------------------------------------------------------- operands
// `box`: rows (K-major) of the operand in a stage, or its columns (panels,
// MN-major); row-major MN-major operands come in 64-column boxes.
bool make_map(CUtensorMap* map, const Operand& o, bool bf16, Form form, uint32_t box) {
  switch (form) {
    case ROWS_K: return make_tmap_rows(map, o.base, bf16, o.planes, o.rows, o.cols, o.ld, o.plane, box, BK, 128);
    case ROWS_MN: return make_tmap_rows(map, o.base, bf16, o.planes, o.rows, o.cols, o.ld, o.plane, BK, 64, 128);
    case PANELS_K: return make_tmap_panels(map, o.base, bf16, o.planes, div_up(o.rows, BM), div_up(o.cols, 8), box, BK / 8);
    default: return make_tmap_panels(map, o.base, bf16, o.planes, div_up(o.rows, BM), div_up(o.cols, 8), BK, box / 8);
  }
}

// ---------------------------------------------------------------- packing
// Copies matrices into operand form: rows padded to 16 bytes, or fp32 values
// as their three bf16 planes.  One launch for all matrices of a call; HBM
// bound (a padded copy moves 4 bytes an element, the planes 10).
struct PackJob {
  const void* src;
  void* dst;
  int64_t rows, cols, ld, plane;
  int64_t first;  // first unit (8 columns of one row) of this job
};
struct PackArgs {
  PackJob job[5];
  int n;
  int64_t units;
};

template <typename T>
__global__ void __launch_bounds__(256) ffn_pack_kernel(const __grid_constant__ PackArgs a) {
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < a.units; u += (int64_t)gridDim.x * 256) {
    int k = 0;
    while (k + 1 < a.n && u >= a.job[k + 1].first) ++k;
    const PackJob& j = a.job[k];
    const int64_t groups = j.ld / 8;
    const int64_t row = (u - j.first) / groups, c0 = ((u - j.first) - row * groups) * 8;
    const T* src = static_cast<const T*>(j.src) + row * j.cols + c0;
    if constexpr (sizeof(T) == 4) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c0 + i < j.cols ? src[i] : 0.0f;
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(j.dst) + row * j.ld + c0;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        __nv_bfloat16 t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t[i] = __float2bfloat16_rn(v[i]);
          const float hi = __bfloat162float(t[i]);
          // inf and NaN are the first plane's alone
          v[i] = fabsf(hi) <= 3.4e38f ? v[i] - hi : 0.0f;
        }
        uint4 w;
        memcpy(&w, t, 16);
        *reinterpret_cast<uint4*>(dst + p * j.plane) = w;
      }
    } else {
      T t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = c0 + i < j.cols ? src[i] : from_f<T>(0.0f);
      uint4 w;
      memcpy(&w, t, 16);
      *reinterpret_cast<uint4*>(static_cast<T*>(j.dst) + row * j.ld + c0) = w;
    }
  }
}

struct Packer {
  PackArgs a{};
  void add(const Operand& o, const void* src) {
    PackJob& j = a.job[a.n];
    j = {src, const_cast<void*>(o.base), o.rows, o.cols, o.ld, o.plane, a.units};
    a.units += o.rows * (o.ld / 8);
    ++a.n;
  }
  template <typename T>
  cudaError_t run(cudaStream_t st) const {
    if (!a.n || !a.units) return cudaSuccess;
    KernelScope ks("ffn_pack", st);
    ffn_pack_kernel<T><<<(unsigned)std::min<int64_t>(div_up(a.units, 256), kSms * 8), 256, 0, st>>>(a);
    return cudaGetLastError();
  }
};

// ---------------------------------------------------------------- split products
// Adds the partials of each cut tile (struct Cut) and stores T.  One CTA per
// 32 x 32 block: warp i adds slots i, i + 8, ... of the tile's list, then the
// eight sums are added in order; reads are whole lines.
struct ReduceArgs {
  const float* partial;
  void* out[2];
  const void* bias;
  int64_t ldo;
  int M, N, base, ctas, vec;  // base: the first cut tile
  GemmArgs g;  // for tile_at, and the cut
};

template <typename T, int BN>
__global__ void __launch_bounds__(256) ffn_reduce_kernel(const __grid_constant__ ReduceArgs a) {
  __shared__ float4 part[8][8][32];
  const int quarters = 4 * a.ctas, blocks = BN / 32 * quarters;  // 32 x 32 blocks of a tile
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x / blocks, blk = blockIdx.x - t * blocks;
  const int q = blk % quarters, c = blk / quarters;
  int z, mt, nt;
  tile_at(a.g, a.base + t, z, mt, nt);
  const int64_t row = (int64_t)mt * BM * a.ctas + q * 32 + lane;
  const int c0 = nt * BN + c * 32;
  if (row - lane >= a.M || c0 >= a.N) return;
  const Cut cut = a.g.cut;
  int run;
  const int n = cut.pieces(t, run);
  float4 v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* first = reinterpret_cast<const float4*>(a.partial + q * (32 * BN) + c * 1024) + lane;
#pragma unroll 2
  for (int i = warp; i < n; i += 8) {
    const float4* p = first + (int64_t)cut.slot(t, i, run) * a.ctas * (BM * BN / 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 f = p[j * 32];
      v[j].x += f.x; v[j].y += f.y; v[j].z += f.z; v[j].w += f.w;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) part[warp][j][lane] = v[j];
  __syncthreads();
  // warp j finishes columns 4 j .. 4 j + 3 of every row
  const int n0 = c0 + 4 * warp;
  if (row >= a.M || n0 >= a.N) return;
  float4 s = part[0][warp][lane];
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    const float4 f = part[w][warp][lane];
    s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
  }
  const float r[4] = {s.x, s.y, s.z, s.w};
  T* out = static_cast<T*>(a.out[z]) + row * a.ldo + n0;
  T o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    o[k] = from_f<T>(r[k] + (a.bias && n0 + k < a.N ? to_f<T>(static_cast<const T*>(a.bias)[n0 + k]) : 0.0f));
  if (a.vec && n0 + 4 <= a.N) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(o[0], o[1], o[2], o[3]);
    else memcpy(__builtin_assume_aligned(out, 8), o, 8);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n0 + k < a.N) out[k] = o[k];
  }
}

// ---------------------------------------------------------------- column sums
// Column sums of dy [M][C] (grad of the down bias): CTA (x, y) adds columns
// 32 VEC x .. of rows y 8 + warp, + 8 gridDim.y, ...; partials [gridDim.y][C].
template <typename T, int VEC>
__global__ void __launch_bounds__(256) ffn_column_partial_kernel(const T* __restrict__ src, float* __restrict__ part,
                                                                 int64_t M, int C) {
  __shared__ float s[8][VEC][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = (blockIdx.x * 32 + lane) * VEC;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  if (c0 < C) {
#pragma unroll 8
    for (int64_t r = (int64_t)blockIdx.y * 8 + warp; r < M; r += (int64_t)gridDim.y * 8) {
      const T* p = src + r * C + c0;
      if constexpr (VEC == 1) {
        acc[0] += to_f<T>(p[0]);
      } else {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        T t[VEC];
        memcpy(t, &w, 16);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += to_f<T>(t[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) s[warp][j][lane] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
    const int l = i / VEC, j = i - l * VEC, c = blockIdx.x * 32 * VEC + i;
    if (c >= C) break;
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += s[w][j][l];
    part[(int64_t)blockIdx.y * C + c] = t;
  }
}

// out[k][c] = sum over the rows of part [rows][sets][N], in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) ffn_column_finish_kernel(const float* __restrict__ part, T* out0, T* out1,
                                                                 int64_t rows, int sets, int N) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, k = blockIdx.y;
  float acc = 0.0f;
  if (c < N) {
#pragma unroll 8
    for (int64_t r = warp; r < rows; r += 32) acc += part[(r * sets + k) * N + c];
  }
  s[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && c < N) {
    float t = 0.0f;
    for (int w = 0; w < 32; ++w) t += s[w][lane];
    T* out = k ? out1 : out0;
    if (out) out[c] = from_f<T>(t);
  }
}

template <typename T, int EPI, int BN, Form A, Form B, bool PAIR>
cudaError_t launch_gemm(const char* name, const Maps& maps, const GemmArgs& a, int workers, cudaStream_t st) {
  auto kern = ffn_gemm_kernel<T, EPI, BN, A, B, PAIR>;
  const int smem = (int)(smem_bytes(EPI, BN, PAIR, sizeof(T) == 4) + kSmemSlack);
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(workers * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(NTHREADS);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 1 : 0;
  KernelScope ks(name, st);
  return cudaLaunchKernelEx(&cfg, kern, maps, a);
}

template <typename T, int EPI, Form A, Form B>
cudaError_t launch_gemm(const char* name, const GemmPlan& p, const Maps& maps, const GemmArgs& a, cudaStream_t st) {
  // pairs have the widest tile of their type, 256 columns or 128 (fp32)
  if (p.pair) return launch_gemm<T, EPI, sizeof(T) == 4 ? 128 : 256, A, B, true>(name, maps, a, p.workers, st);
  switch (p.bn) {
    case 256:
      if constexpr (sizeof(T) == 2) return launch_gemm<T, EPI, 256, A, B, false>(name, maps, a, p.workers, st);
      return cudaErrorInvalidValue;  // fp32 plans stop at 128
    case 128: return launch_gemm<T, EPI, 128, A, B, false>(name, maps, a, p.workers, st);
    default: return launch_gemm<T, EPI, 64, A, B, false>(name, maps, a, p.workers, st);
  }
}

// Segments of products of the given (a map, b map) pairs.
template <typename T>
int fill_segments(Seg* seg, const std::vector<std::pair<int, int>>& pairs) {
  static const int kOrder[6][2] = {{0, 2}, {1, 1}, {2, 0}, {0, 1}, {1, 0}, {0, 0}};
  int n = 0;
  if (sizeof(T) == 4) {
    for (auto& o : kOrder)
      for (auto& p : pairs) seg[n++] = {(uint8_t)p.first, (uint8_t)o[0], (uint8_t)p.second, (uint8_t)o[1]};
  } else {
    for (auto& p : pairs) seg[n++] = {(uint8_t)p.first, 0, (uint8_t)p.second, 0};
  }
  return n;
}

// Rows of the row operand in a stage, and what the kernel is told of them
// (GemmArgs): a tile's 128, or with one row tile those that exist.
uint32_t row_box(GemmArgs& a, const GemmPlan& p, Form form, Form columns) {
  a.cols = p.cols;
  uint32_t rows = BM;
  if (!p.pair && p.tiles_m == 1 && columns == ROWS_K) {
    if (form == PANELS_K) rows = (uint32_t)round_up(a.M, 32);
    if (form == ROWS_K) rows = (uint32_t)round_up(a.M, 8);
  }
  a.a_bytes = rows * 128;
  a.a_lbo = rows * 16;
  return rows;
}

template <typename T>
constexpr bool operand_bf16() { return !std::is_same<T, __half>::value; }

// A product with plain sums as its result: out[z] = sum of the segments (+ bias).
// a[z], z < batches: the row operands (one batch), or with one batch the row
// operands of the pairs; b: the column operands of the pairs.
template <typename T, Form A, Form B>
cudaError_t store_product(const char* name, const std::vector<Operand>& a_ops, const std::vector<Operand>& b_ops,
                          int64_t M, int64_t N, int64_t K, int batches, void* const* out, int64_t ldo,
                          const void* bias, float* partial, cudaStream_t st) {
  const int pairs = (int)b_ops.size();
  Maps maps;
  GemmArgs a{};
  std::vector<std::pair<int, int>> pl;
  const int n_a = (int)a_ops.size();
  for (int i = 0; i < pairs; ++i) pl.push_back({i, n_a + i});
  a.nseg = fill_segments<T>(a.seg, pl);
  a.M = (int)M; a.N = (int)N;
  a.nk = (int)div_up(K, BK);
  const GemmPlan p = plan_gemm(M, N, (int64_t)a.nk * a.nseg, batches, false, true, sizeof(T) == 4, B == ROWS_K);
  for (int i = 0; i < n_a; ++i)
    if (!make_map(&maps.m[i], a_ops[i], operand_bf16<T>(), A, row_box(a, p, A, B))) return cudaErrorInvalidValue;
  for (int i = 0; i < pairs; ++i)
    if (!make_map(&maps.m[n_a + i], b_ops[i], operand_bf16<T>(), B, (uint32_t)(p.pair ? p.bn / 2 : p.cols)))
      return cudaErrorInvalidValue;
  set_tiles(a, p.tiles_m, p.tiles_n, batches);
  a.split = p.split;
  a.cut = p.cut;
  a.operand_bf16 = operand_bf16<T>();
  a.partial = partial;
  a.out[0] = out[0];
  a.out[1] = batches > 1 ? out[1] : nullptr;
  a.ldo = ldo;
  a.vec = (ldo * (int64_t)sizeof(T)) % 16 == 0;
  for (int z = 0; z < batches; ++z) a.vec = a.vec && (reinterpret_cast<uintptr_t>(out[z]) & 15) == 0;
  if (sizeof(T) == 2 && a.vec)
    for (int z = 0; z < batches; ++z)
      if (!make_tmap_rows(&maps.out[z], out[z], operand_bf16<T>(), 1, M, N, ldo, M * ldo, 32, (uint32_t)(p.bn / 4), p.bn / 2))
        return cudaErrorInvalidValue;
  a.bias[0] = bias;
  cudaError_t e = tc_status_ptr(&a.status);
  if (e != cudaSuccess) return e;
  if ((e = launch_gemm<T, EPI_STORE, A, B>(name, p, maps, a, st)) != cudaSuccess || !p.split) return e;
  ReduceArgs r{};
  r.partial = partial;
  r.out[0] = a.out[0]; r.out[1] = a.out[1];
  r.bias = bias;
  r.ldo = ldo;
  r.M = a.M; r.N = a.N; r.g = a;
  r.vec = a.vec;
  r.base = p.tiles_m * p.tiles_n * batches - p.cut.R;
  KernelScope ks("ffn_reduce", st);
  r.ctas = p.pair ? 2 : 1;
  const unsigned grid = (unsigned)(p.cut.R * (p.bn / 32 * 4 * r.ctas));
  if (p.bn == 256) ffn_reduce_kernel<T, 256><<<grid, 256, 0, st>>>(r);
  else if (p.bn == 128) ffn_reduce_kernel<T, 128><<<grid, 256, 0, st>>>(r);
  else ffn_reduce_kernel<T, 64><<<grid, 256, 0, st>>>(r);
  return cudaGetLastError();
}

template <typename T>
cudaError_t forward_t(const FfnProblem& p, const FfnTensors& t, void* y, void* saved, void* ws, cudaStream_t st) {
  const Shape s(p);
  void* hidden = saved ? static_cast<uint8_t*>(saved) + s.blocks_bytes() : nullptr;
  const ForwardWs w(p, t, ws, hidden);
  if (w.few) {
    const FewArgs up{t.x, {t.w_gate, t.w_up}, {t.b_gate, t.b_up}, w.few, (int)s.M, (int)s.F, (int)s.C, p.act};
    const FewArgs down{w.few, {t.w_down, nullptr}, {t.b_down, nullptr}, y, (int)s.M, (int)s.C, (int)s.F, p.act};
    const cudaError_t e = launch_few<T, true>("ffn_few_gate_up", up, st);
    return e != cudaSuccess ? e : launch_few<T, false>("ffn_few_down", down, st);
  }
  Packer pk;
  if (w.pack_c) {
    pk.add(w.x, t.x);
    pk.add(w.wg, t.w_gate);
    pk.add(w.wu, t.w_up);
  }
  if (w.pack_f) pk.add(w.wd, t.w_down);
  cudaError_t e = pk.run<T>(st);
  if (e != cudaSuccess) return e;

  GemmArgs a{};
  Maps maps;
  a.nseg = fill_segments<T>(a.seg, {{0, 1}});
  a.M = (int)s.M; a.N = (int)s.F;
  a.nk = (int)div_up(s.C, BK);
  const GemmPlan plan = plan_gemm(s.M, s.F, (int64_t)a.nk * a.nseg, 1, true, false, sizeof(T) == 4, true);
  if (!make_map(&maps.m[0], w.x, operand_bf16<T>(), ROWS_K, row_box(a, plan, ROWS_K, ROWS_K)) ||
      !make_map(&maps.m[1], w.wg, operand_bf16<T>(), ROWS_K, (uint32_t)plan.cols) ||
      !make_map(&maps.m[2], w.wu, operand_bf16<T>(), ROWS_K, (uint32_t)plan.cols))
    return cudaErrorInvalidValue;
  set_tiles(a, plan.tiles_m, plan.tiles_n, 1);
  a.act = p.act;
  a.operand_bf16 = operand_bf16<T>();
  a.out[0] = const_cast<void*>(w.h.base);
  a.ldo = div_up(s.F, 8);
  a.plane = s.panel_plane_bytes();
  a.bias[0] = t.b_gate; a.bias[1] = t.b_up;
  a.saved = s.recompute() ? nullptr : saved;
  if ((e = tc_status_ptr(&a.status)) != cudaSuccess) return e;
  if ((e = launch_gemm<T, EPI_GATED, ROWS_K, ROWS_K>("ffn_gate_up", plan, maps, a, st)) != cudaSuccess || !y) return e;
  return store_product<T, PANELS_K, ROWS_K>("ffn_down", {w.h}, {w.wd}, s.M, s.C, s.F, 1, &y, s.C, t.b_down, w.partial, st);
}

template <typename T>
cudaError_t backward_t(const FfnProblem& p, const FfnTensors& t, const void* dy, const void* saved, const FfnGrads& g,
                       void* ws, cudaStream_t st, dcn_params_ready_fn ready, void* user) {
  const Shape s(p);
  const BackwardWs w(p, t, dy, ws);
  const Operand h = s.operand(static_cast<const uint8_t*>(saved) + s.blocks_bytes(), s.M, s.F);  // panels
  Packer pk;
  if (w.pack_c) {
    pk.add(w.x, t.x);
    pk.add(w.dy, dy);
    pk.add(w.wg, t.w_gate);
    pk.add(w.wu, t.w_up);
  }
  if (w.pack_f) pk.add(w.wd, t.w_down);
  cudaError_t e = pk.run<T>(st);
  if (e != cudaSuccess) return e;

  const bool hidden_grads = g.x || g.w_gate || g.w_up || g.b_gate || g.b_up;
  if (hidden_grads) {
    GemmArgs a{};
    Maps maps;
    const bool again = s.recompute(), bf16 = operand_bf16<T>();
    a.nseg = fill_segments<T>(a.seg, {{0, again ? 2 : 1}});
    a.M = (int)s.M; a.N = (int)s.F;
    a.nk = (int)div_up(s.C, BK);
    GemmPlan plan = plan_gemm(s.M, s.F, (int64_t)a.nk * a.nseg, 1, false, false, sizeof(T) == 4, false);
    bool ok;
    if (again) {
      plan.pair = false;
      plan.tiles_m = (int)div_up(s.M, BM);
      plan.tiles_n = (int)div_up(s.F, kRecomputeCols);
      plan.workers = (int)std::min<int64_t>((int64_t)plan.tiles_m * plan.tiles_n, kSms);
      ok = make_map(&maps.m[0], w.x, bf16, ROWS_K, BM) && make_map(&maps.m[1], w.dy, bf16, ROWS_K, BM) &&
           make_map(&maps.m[2], w.wg, bf16, ROWS_K, kRecomputeCols) &&
           make_map(&maps.m[3], w.wu, bf16, ROWS_K, kRecomputeCols) && make_map(&maps.m[4], w.wd, bf16, ROWS_MN, BK);
      a.bias[0] = t.b_gate; a.bias[1] = t.b_up;
    } else {
      ok = make_map(&maps.m[0], w.dy, bf16, ROWS_K, BM) && make_map(&maps.m[1], w.wd, bf16, ROWS_MN, BK);
      a.saved = const_cast<void*>(saved);
    }
    if (!ok) return cudaErrorInvalidValue;
    set_tiles(a, plan.tiles_m, plan.tiles_n, 1);
    a.act = p.act;
    a.operand_bf16 = bf16;
    a.out[0] = const_cast<void*>(w.dg.base); a.out[1] = const_cast<void*>(w.du.base);
    a.ldo = div_up(s.F, 8);
    a.plane = s.panel_plane_bytes();
    a.colsum = g.b_gate || g.b_up ? w.colsum : nullptr;
    if ((e = tc_status_ptr(&a.status)) != cudaSuccess) return e;
    e = again ? launch_gemm<T, EPI_RECOMPUTE, kRecomputeBn, ROWS_K, ROWS_K, false>("ffn_dhidden", maps, a, plan.workers, st)
              : launch_gemm<T, EPI_DGATE, ROWS_K, ROWS_MN>("ffn_dhidden", plan, maps, a, st);
    if (e != cudaSuccess) return e;
    if (a.colsum) {
      KernelScope ks("ffn_column_finish", st);
      ffn_column_finish_kernel<T><<<dim3((unsigned)div_up(s.F, 32), 2), 1024, 0, st>>>(
          w.colsum, static_cast<T*>(g.b_gate), static_cast<T*>(g.b_up), (int64_t)plan.tiles_m * (plan.pair ? 8 : 4), 2, (int)s.F);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
  }
  if (g.w_down &&
      (e = store_product<T, ROWS_MN, PANELS_MN>("ffn_dw_down", {w.dy}, {h}, s.C, s.F, s.M, 1, &g.w_down, s.F, nullptr, w.partial, st)) !=
          cudaSuccess)
    return e;
  if (g.w_gate && g.w_up) {
    void* const out[2] = {g.w_gate, g.w_up};
    e = store_product<T, PANELS_MN, ROWS_MN>("ffn_dw_gate_up", {w.dg, w.du}, {w.x}, s.F, s.C, s.M, 2, out, s.C, nullptr, w.partial, st);
  } else if (g.w_gate || g.w_up) {
    void* const out[1] = {g.w_gate ? g.w_gate : g.w_up};
    e = store_product<T, PANELS_MN, ROWS_MN>("ffn_dw_gate_up", {g.w_gate ? w.dg : w.du}, {w.x}, s.F, s.C, s.M, 1, out, s.C, nullptr,
                                     w.partial, st);
  }
  if (e != cudaSuccess) return e;
  if (g.b_down) {
    constexpr int kVec = 16 / sizeof(T);
    const int64_t rows = std::min<int64_t>(div_up(s.M, 64), kSumSlices);
    {
      KernelScope ks("ffn_column_partial", st);
      if (s.C % kVec == 0)
        ffn_column_partial_kernel<T, kVec><<<dim3((unsigned)div_up(s.C, 32 * kVec), (unsigned)rows), 256, 0, st>>>(
            static_cast<const T*>(dy), w.rowsum, s.M, (int)s.C);
      else
        ffn_column_partial_kernel<T, 1><<<dim3((unsigned)div_up(s.C, 32), (unsigned)rows), 256, 0, st>>>(
            static_cast<const T*>(dy), w.rowsum, s.M, (int)s.C);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    KernelScope ks("ffn_column_finish", st);
    ffn_column_finish_kernel<T><<<dim3((unsigned)div_up(s.C, 32), 1), 1024, 0, st>>>(
        w.rowsum, static_cast<T*>(g.b_down), nullptr, rows, 1, (int)s.C);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if (ready) ready(user);
  if (!g.x) return cudaSuccess;
  return store_product<T, PANELS_K, ROWS_MN>("ffn_dx", {w.dg, w.du}, {w.wg, w.wu}, s.M, s.C, s.F, 1, &g.x, s.C, nullptr, w.partial, st);
}

}  // namespace

// The two passes of one data type, for dcn_ffn.cu.
#define DCN_FFN_INSTANTIATE(T, name)                                                                              \
  cudaError_t ffn_forward_##name(const FfnProblem& p, const FfnTensors& t, void* y, void* saved, void* workspace, \
                                 cudaStream_t st) {                                                               \
    return forward_t<T>(p, t, y, saved, workspace, st);                                                           \
  }                                                                                                               \
  cudaError_t ffn_backward_##name(const FfnProblem& p, const FfnTensors& t, const void* dy, const void* saved,    \
                                  const FfnGrads& g, void* workspace, cudaStream_t st, dcn_params_ready_fn ready, \
                                  void* user) {                                                                   \
    return backward_t<T>(p, t, dy, saved, g, workspace, st, ready, user);                                         \
  }

}  // namespace dcn
