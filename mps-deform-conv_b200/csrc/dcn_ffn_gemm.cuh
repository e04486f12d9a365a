// dcn_ffn_gemm.cuh -- the matrix products of the gated feed-forward block on
// tcgen05, with the block's elementwise work in their epilogues.
//
//   D[m][n] = sum over segments s, sum over k of A_s(m, k) B_s(n, k)
//
// A segment names the tensor map and plane of each operand.  16-bit data is
// one plane.  fp32 data is held as three bf16 planes, v = p0 + p1 + p2 exactly
// to 24 bits (each plane the rounding of what the ones before left), and a
// product takes the six segments whose terms are not below 2^-24 of it:
//   p0 p2, p1 p1, p2 p0, p0 p1, p1 p0, p0 p0          (smallest terms first)
// which cost as much as three tf32 passes, keep every bit and need no
// transposed copies: 16-bit operands may be MN-major, tf32 ones may not.
//
// Either operand may be K-major (rows of the contracted axis, "x W^T") or
// MN-major (rows of the output axis, "dgate^T x"): TMA fetches 64 contracted
// values a stage in either form, zero-filled past the tensors' ends, so no
// size needs to be a multiple of anything.
//
// The caller's matrices are row-major (128-byte-swizzled tiles).  The block's
// own operands (hidden, dgate, dup) lie in panels: of each 128 rows, panel p
// holds columns 8 p .. 8 p + 7, 16 bytes a row, and the panels of the 128 rows
// follow one another (a tile is one run of memory).  The lanes of an epilogue
// warp are rows, so they store 512 contiguous bytes an instruction from their
// registers, where a row-major matrix needs staging in shared memory, a proxy
// fence and TMA stores with short rows (measured: gate and up of 92416 x 512 ->
// 2048 in bf16 437 -> 402 us, dhidden of 921600 x 64 -> 170 in fp16 249 -> 217,
// of 8192 x 128 -> 512 in fp32 66 -> 46).  Eight rows of a panel are 128
// contiguous bytes, the matrix unit's 8 x 16-byte core matrix without swizzle,
// read K-major or MN-major as a product needs it.
//
// Warp roles (640 threads): warps 0-15 epilogue, warp 16 issues the MMAs, warp
// 17 the TMA loads.  A CTA works through its share of the output tiles; the
// accumulator is double-buffered in TMEM, so a tile's epilogue runs under the
// next tile's MMAs.  Epilogue warp w reads TMEM lanes 32 (w % 4) .. +31: lane i
// owns one row, 16 columns at a time, and takes blocks w / 4, w / 4 + 4, ... of
// the tile.  A block's sums are read while the one before is worked on, and the
// buffer goes back to the MMAs once the last has been read; held to the end of
// the epilogue, a buffer's products and its epilogue would exclude each other.
//
// What bounds it: products with a long K the tensor cores, at 1.3 to 1.45
// PFLOP/s in bf16 until the power cap is reached.  Gated passes the epilogue: 35
// instructions a value pair, issued by four warps a scheduler that wait for
// TMEM and for one another's results in between.  23104 x 512 -> 2048 in bf16:
// a pair of tiles every 8000 cycles, in 4100 of which the tensor cores work;
// issue slots 55 % (gate and up) and 56 % (dhidden) busy, tensor cores 51 and
// 23 %.  27200 x 256 -> 1024: 42 us with relu, 53 with gelu, 18 us of operations
// at the measured matrix rate.  Arithmetic in packed pairs (f32x2), not used
// here, gained 2 % where gate and up are 92416 x 512 -> 2048 (419 us against 428;
// forward and backward 1742 against 1752) and nothing in that case (both products
// 81.2 us both ways), timed while the cut's state still took registers here.
//
// Work is dealt in whole tiles: worker w takes tiles w, w + W, ...  Where the
// last wave would leave many of the W workers idle, its R tiles are cut along
// K instead (struct Cut): up to W / R workers a tile walk slices of K of one
// length, tile by tile side by side, so that at any time all tiles read the same
// rows of both operands and these come from the L2 (dealt tile after tile, a
// product with a long K reads them from memory once per tile); workers left
// over share the end of K in runs no longer than a slice.  Each piece is an fp32
// partial in a slot of its own, and a second kernel adds a tile's slots in a
// fixed order: the result does not depend on timing.
//
// Pairs (template PAIR): two CTAs of a cluster share a tile of 256 rows
// (tcgen05 cta_group::2).  Each holds its own 128 rows of the row operand, half
// of the column operand (GATED: one gate, the other up) and the accumulator of
// its rows; the first issues the MMAs for both.  A CTA alone reads 384 operand
// rows for 128 x 256 results, a pair 512 for 256 x 256, a third less (92416 x 512
// -> 2048 in bf16: dx 284 -> 266 us, weight gradients 446 -> 413).  Loads go to
// the CTA's own shared memory and report to the first CTA's barrier; commits
// arrive at both.
//
// Every mbarrier wait is bounded (dcn_sm100.cuh).
#pragma once

#include <cuda.h>

#include <type_traits>

#include "dcn_common.cuh"
#include "dcn_ffn_layout.h"
#include "dcn_sm100.cuh"
#include "dcn_tc_common.cuh"

namespace dcn {
namespace ffn {

using namespace sm100;

constexpr int kActSilu = DCN_ACT_SILU, kActGelu = DCN_ACT_GELU, kActRelu = DCN_ACT_RELU, kActSigmoid = DCN_ACT_SIGMOID;

constexpr int EPI_WARPS = 16;
constexpr int MMA_WARP = EPI_WARPS, LOAD_WARP = EPI_WARPS + 1;
constexpr int NTHREADS = (EPI_WARPS + 4) * 32;  // whole warpgroups: two warps of the last idle
// Registers: 640 threads start with 96 each (61,440); the epilogue warps take
// what the last warpgroup gives up: 512 x 112 + 128 x 32 = 61,440.
constexpr int kEpiRegs = 112, kOtherRegs = 32;
constexpr int CB = 16;           // columns of an epilogue block
constexpr uint32_t A_STAGE = BM * 128;
constexpr int ST_FFN_LOAD = 61, ST_FFN_MMA = 62, ST_FFN_EPI = 63, ST_FFN_DRAIN = 64, ST_FFN_SMEM = 65;

enum Epi { EPI_GATED, EPI_DGATE, EPI_RECOMPUTE, EPI_STORE };

// Accumulator columns are BN; EPI_RECOMPUTE has 3 x 64 (gate, up, dhidden) and
// two row operands (x, dy).
constexpr int kRecomputeCols = 64, kRecomputeBn = 3 * kRecomputeCols;
// Output staging of an epilogue warp: STORE (16-bit) its columns of a tile for
// one TMA store, DGATE and RECOMPUTE an fp32 block whose columns are summed.
constexpr uint32_t kSumBlock = 32 * CB * 4;
__host__ __device__ constexpr uint32_t staging_bytes(int epi, int bn, bool wide) {
  return wide || epi == EPI_GATED ? 0u : epi == EPI_STORE ? 32u * (uint32_t)(bn / 4) * 2u : kSumBlock;
}
__host__ __device__ constexpr uint32_t stage_bytes(int bn, bool pair) {
  return (bn == kRecomputeBn ? 2 : 1) * A_STAGE + (uint32_t)bn * 128u / (pair ? 2u : 1u);
}
constexpr uint32_t kBiasBytes = EPI_WARPS * 32 * 4u, kBarBytes = 256;
// dynamic shared memory starts on 1024 bytes when a kernel has no static one;
// this much is left over for a start that does not (checked by the kernel)
constexpr uint32_t kSmemSlack = 512;
// as many stages as fit, at most eight
__host__ __device__ constexpr int stages(int epi, int bn, bool pair, bool wide) {
  const uint32_t n = (232448u - kSmemSlack - kBiasBytes - kBarBytes - EPI_WARPS * staging_bytes(epi, bn, wide)) /
                     stage_bytes(bn, pair);
  return n < 8 ? (int)n : 8;
}
__host__ __device__ constexpr uint32_t smem_bytes(int epi, int bn, bool pair, bool wide) {
  return (uint32_t)stages(epi, bn, pair, wide) * stage_bytes(bn, pair) + EPI_WARPS * staging_bytes(epi, bn, wide) +
         kBiasBytes + kBarBytes;
}
// fp32 data: K blocks added up in TMEM before their sum moves on to registers
constexpr int kWideRun = 4;

// n / d for 0 <= n < 2^31 by a multiplication: mul = ceil(2^(31 + s) / d) with
// 2^s >= d, so the rounding adds less than n / 2^31 to the quotient times 2^s / d.
struct FastDiv {
  uint32_t mul, shift, d;
  __host__ __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
#ifdef __CUDA_ARCH__
    return d == 1 ? n : __umulhi(n, mul) >> shift;
#else
    return n / d;
#endif
  }
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  const uint64_t p = uint64_t(1) << (31 + s);
  return {(uint32_t)((p + d - 1) / d), s ? s - 1 : 0, d};
}
constexpr int kGroupM = 8;

struct Seg {
  uint8_t a_map, a_plane, b_map, b_plane;
};
struct Maps {
  CUtensorMap m[5];
  CUtensorMap out[2];  // STORE, 16-bit: 32 rows x a warp's columns
};

struct GemmArgs {
  int M, N;                  // output extents (GATED, DGATE: N = F)
  int nk, nseg;              // K blocks of a segment, segments
  Seg seg[12];
  int tiles_m, tiles_n, batches;  // a batch adds its index to a_map (and picks the output)
  // tiles are dealt in blocks of kGroupM row tiles x all column tiles; divisors of tile_at
  FastDiv per_batch, per_block, last_rows;
  int split;                 // 1: the last cut.R tiles are cut along K, partials to `partial`
  Cut cut;
  int act;
  // GATED, and STORE of ROWS_K columns, without pairs: output columns of a tile (a
  // multiple of 16, at most the kernel's), bytes of the row operand in a stage and
  // (panels) between its panels there.  With one row tile only the rows that exist
  // are loaded; what the others hold is multiplied into results that are not stored.
  int cols;
  uint32_t a_bytes, a_lbo;
  uint32_t operand_bf16;
  float* partial;
  // outputs: STORE: out[batch] [M][ldo] of T (+ bias); else panels of hidden, or dgate and dup:
  // ldo panels of 128 rows, `plane` bytes between the bf16 planes of fp32 data
  void* out[2];
  int64_t ldo, plane;
  int vec;                   // out rows take 16-byte stores (16-bit data: TMA stores)
  const void* bias[2];       // STORE: [0]; GATED, RECOMPUTE: gate, up
  void* saved;               // gate and up (private layout, below), or null
  float* colsum;             // DGATE: [32-row block][2][F] column sums of dgate and dup, or null
  int* status;
};

// ---------------------------------------------------------------- saved gate / up
// What the backward needs of a 32-row x 16-column block (its rows being the
// lanes of one warp) lies together, each 16-byte piece of the 32 lanes side by
// side, so both passes move whole lines:
//   16-bit data: gate, up as fp16: 11 bits, not bf16's 8, of values that the
//     derivative multiplies, at the same size.  A row whose largest value of the
//     16 columns is outside [2^-4, 2^15) is multiplied by powers of two that bring
//     the largest below 2^15.  One int16 per lane holds the two exponents (14: as
//     they are); a warp without such a row skips the scaling;
//   fp32 data: gate, up as fp32.
template <typename T>
__host__ __device__ inline size_t saved_block_offset(int64_t m_block, int64_t col_block, int64_t col_blocks) {
  return (size_t)(m_block * col_blocks + col_block) * saved_block_bytes(sizeof(T) == 4);
}

__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&v)[CB]) {
  uint32_t r[CB];
  tmem_ld16(taddr, r);
#pragma unroll
  for (int i = 0; i < CB; ++i) v[i] = __uint_as_float(r[i]);
}
// Waits for this warp's TMEM loads; the values pass through, so that nothing
// that uses them is scheduled before the wait.
__device__ __forceinline__ void tmem_wait(float (&v)[CB]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Descriptor of an operand in panels: core matrices of 8 rows x 16 bytes without
// swizzle; lbo, sbo as the operand's major asks (bytes).
__device__ __forceinline__ uint64_t desc_panels(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;
  return d;
}

// ---------------------------------------------------------------- CTA pairs
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// All threads of both CTAs.
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The cluster address of `addr` in the first CTA.
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// Relaxed: what the arrival publishes is that TMEM has been read (tcgen05 fence
// before it); a release would wait for all of the thread's stores to global
// memory (2100 cycles a tile).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc_g(uint32_t slot, uint32_t ncols) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(slot, ncols);
    tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc_g(uint32_t taddr, uint32_t ncols) {
  if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
  else tmem_dealloc(taddr, ncols);
}
template <bool PAIR>
__device__ __forceinline__ void mma_g(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    mma_f16(d, ad, bd, idesc, accumulate);
}
// Arrives on `bar` of this CTA (PAIR and both: of both CTAs) once the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit_g(uint32_t bar, bool both) {
  if (!PAIR) {
    mma_commit(bar);
  } else if (both) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  }
}
// A load into this CTA's shared memory; PAIR: `bar` is a cluster address in the first CTA.
template <bool PAIR>
__device__ __forceinline__ void load_g(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    tma_load_3d(dst, map, x, y, z, bar);
}

// The same for panels: boxes of 512-byte pieces (32 rows of a panel).
template <bool PAIR>
__device__ __forceinline__ void load_panels(uint32_t dst, const CUtensorMap* map, int row, int panel, int plane,
                                            uint32_t bar) {
  const int piece = (row >> 5) & 3, rows = row >> 7;
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(piece), "r"(panel), "r"(rows), "r"(plane), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(piece), "r"(panel), "r"(rows), "r"(plane), "r"(bar)
        : "memory");
}

// ---------------------------------------------------------------- activations
// ACCURATE (fp32 data): CUDA's expf, normcdff and IEEE division.  Else the matching
// hardware approximations, whose few ulp are far below a 16-bit result's
// rounding, with subnormals flushed (an exponential below 2^-126 is 0 here;
// the forms that keep them cost four instructions more each).
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
template <bool ACCURATE>
__device__ __forceinline__ float sigmoid(float x) {
  // far below zero the exponential overflows to inf and the quotient is 0, as it should be
  return ACCURATE ? 1.0f / (1.0f + expf(-x)) : rcp_fast(1.0f + exp2_fast(-kLog2e * x));
}
// The normal distribution function and exp(-x^2 / 2).  fp32: not 1 + erf(x / sqrt 2),
// which cancels in the lower tail (at -5 a tenth of the value, below -5.5 all of it;
// normcdff is within 5 ulp).  Fast form: with z = |x|,
// Phi(-z) = exp(-z^2 / 2) R(z), where R(z) = erfcx(z / sqrt 2) / 2 is smooth and
// R ~ t (c0 + c1 t + ... + c5 t^5), t = 1 / (1 + 0.308 z): coefficients fitted
// here for the least largest relative error, 4e-6 over z in [0, 14] (past that
// the exponential is 0).  Both tails keep that relative error, and the
// derivative needs the same exponential.
template <bool ACCURATE>
__device__ __forceinline__ float2 normal_cdf(float x) {
  if (ACCURATE) return make_float2(normcdff(x), expf(-0.5f * x * x));
  const float z = fabsf(x);
  const float t = rcp_fast(fmaf(0.308f, z, 1.0f));
  const float e = exp2_fast((-0.5f * kLog2e) * (z * z));
  float r = fmaf(t, -0.0754310913f, 0.189621131f);
  r = fmaf(t, r, 0.00726954421f);
  r = fmaf(t, r, 0.136535319f);
  r = fmaf(t, r, 0.118880802f);
  r = fmaf(t, r, 0.123122739f);
  const float low = e * (t * r);
  return make_float2(x > 0.0f ? 1.0f - low : low, e);
}
template <bool ACCURATE, int ACT>
__device__ __forceinline__ float act_value(float x) {
  if constexpr (ACT == kActSilu) return x * sigmoid<ACCURATE>(x);
  else if constexpr (ACT == kActGelu) return x * normal_cdf<ACCURATE>(x).x;
  else if constexpr (ACT == kActRelu) return x > 0.0f ? x : (x == x ? 0.0f : x);
  else return sigmoid<ACCURATE>(x);
}
// act(x) and act'(x)
template <bool ACCURATE, int ACT>
__device__ __forceinline__ float2 act_both(float x) {
  if constexpr (ACT == kActSilu) {
    const float s = sigmoid<ACCURATE>(x), a = x * s;
    return make_float2(a, fmaf(a, 1.0f - s, s));
  } else if constexpr (ACT == kActGelu) {
    const float2 c = normal_cdf<ACCURATE>(x);
    return make_float2(x * c.x, fmaf(x, 0.39894228040143268f * c.y, c.x));
  } else if constexpr (ACT == kActRelu) {
    return x > 0.0f ? make_float2(x, 1.0f) : make_float2(x == x ? 0.0f : x, 0.0f);
  } else {
    const float s = sigmoid<ACCURATE>(x);
    return make_float2(s, s * (1.0f - s));
  }
}
// A row's block at a time; the activation is picked once for all of it.
template <bool ACCURATE, int ACT>
__device__ __forceinline__ void gate_block(const float (&g)[CB], const float (&u)[CB], float (&h)[CB]) {
#pragma unroll
  for (int j = 0; j < CB; ++j) h[j] = act_value<ACCURATE, ACT>(g[j]) * u[j];
}
// (gate, up) to (dgate, dup)
template <bool ACCURATE, int ACT>
__device__ __forceinline__ void dgate_block(const float (&dh)[CB], float (&g)[CB], float (&u)[CB]) {
#pragma unroll
  for (int j = 0; j < CB; ++j) {
    const float2 s = act_both<ACCURATE, ACT>(g[j]);
    g[j] = dh[j] * u[j] * s.y;
    u[j] = dh[j] * s.x;
  }
}
template <bool ACCURATE>
__device__ __forceinline__ void gate_block(int act, const float (&g)[CB], const float (&u)[CB], float (&h)[CB]) {
  if (act == kActSilu) gate_block<ACCURATE, kActSilu>(g, u, h);
  else if (act == kActGelu) gate_block<ACCURATE, kActGelu>(g, u, h);
  else if (act == kActRelu) gate_block<ACCURATE, kActRelu>(g, u, h);
  else gate_block<ACCURATE, kActSigmoid>(g, u, h);
}
template <bool ACCURATE>
__device__ __forceinline__ void dgate_block(int act, const float (&dh)[CB], float (&g)[CB], float (&u)[CB]) {
  if (act == kActSilu) dgate_block<ACCURATE, kActSilu>(dh, g, u);
  else if (act == kActGelu) dgate_block<ACCURATE, kActGelu>(dh, g, u);
  else if (act == kActRelu) dgate_block<ACCURATE, kActRelu>(dh, g, u);
  else dgate_block<ACCURATE, kActSigmoid>(dh, g, u);
}

// ---------------------------------------------------------------- stores
__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// values 8 j .. 8 j + 7 of a block as 16-bit
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[CB], int j) {
  uint4 p;
  p.x = pack2(v[8 * j], v[8 * j + 1], (T*)nullptr);
  p.y = pack2(v[8 * j + 2], v[8 * j + 3], (T*)nullptr);
  p.z = pack2(v[8 * j + 4], v[8 * j + 5], (T*)nullptr);
  p.w = pack2(v[8 * j + 6], v[8 * j + 7], (T*)nullptr);
  return p;
}
// the same times s
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[CB], int j, float s) {
  uint4 p;
  p.x = pack2(v[8 * j] * s, v[8 * j + 1] * s, (T*)nullptr);
  p.y = pack2(v[8 * j + 2] * s, v[8 * j + 3] * s, (T*)nullptr);
  p.z = pack2(v[8 * j + 4] * s, v[8 * j + 5] * s, (T*)nullptr);
  p.w = pack2(v[8 * j + 6] * s, v[8 * j + 7] * s, (T*)nullptr);
  return p;
}

// A block's columns of one row of a row-major matrix of T with `n` columns.
template <typename T>
__device__ __forceinline__ void store_row(T* row, int c0, int n, bool vec, const float (&v)[CB]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < CB / 4; ++j)
        if (c0 + 4 * j < n)
          *reinterpret_cast<float4*>(row + c0 + 4 * j) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < CB / 8; ++j)
        if (c0 + 8 * j < n) *reinterpret_cast<uint4*>(row + c0 + 8 * j) = pack8<T>(v, j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < CB; ++j)
      if (c0 + j < n) row[c0 + j] = from_f<T>(v[j]);
  }
}

// A block's two 16-byte pieces of a staged row of W bytes, with the swizzle of
// that width (128, 64 or 32 bytes: piece j of row r at j ^ (r % 8), j ^ (r / 2 %
// 4) or j ^ (r / 4 % 2)), so eight lanes cover all banks.
template <int W>
__device__ __forceinline__ uint32_t staged_piece(int row, int j) {
  return row * W + ((W == 128 ? j ^ (row & 7) : W == 64 ? j ^ ((row >> 1) & 3) : j ^ ((row >> 2) & 1)) << 4);
}
template <typename T, int W>
__device__ __forceinline__ void stage_row(uint8_t* rows, int lane, int block, const float (&v)[CB]) {
#pragma unroll
  for (int j = 0; j < CB / 8; ++j)
    *reinterpret_cast<uint4*>(rows + staged_piece<W>(lane, 2 * block + j)) = pack8<T>(v, j);
}
// 32 rows of a warp's columns leave in one TMA store; rows and columns past the
// matrix are dropped by it.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(z), "r"(src)
               : "memory");
}

// A block's columns of one row, as an operand of a following product: two
// panels' pieces (fp32 data: in each of three bf16 planes).  `at`: this row in
// the first panel, 2048 bytes before the next; a panel at or past column `left`
// is not in the matrix and is skipped (a last panel's other columns are zero).
template <typename T>
__device__ __forceinline__ void store_panels(uint8_t* at, int64_t plane, int left, const float (&v)[CB]) {
  constexpr int kPanel = BM * 16;
  if constexpr (sizeof(T) == 4) {
    float r[CB];
#pragma unroll
    for (int j = 0; j < CB; ++j) r[j] = v[j];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
#pragma unroll
      for (int j = 0; j < CB / 8; ++j)
        if (8 * j < left) *reinterpret_cast<uint4*>(at + k * plane + j * kPanel) = pack8<__nv_bfloat16>(r, j);
      // a plane that holds inf or NaN ends the expansion: the others are zero
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        const float hi = __bfloat162float(__float2bfloat16_rn(r[j]));
        r[j] = fabsf(hi) <= 3.4e38f ? r[j] - hi : 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < CB / 8; ++j)
      if (8 * j < left) *reinterpret_cast<uint4*>(at + j * kPanel) = pack8<T>(v, j);
  }
}

// ---------------------------------------------------------------- saved values
__device__ __forceinline__ float largest(const float (&v)[CB]) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < CB; ++j) top = fmaxf(top, fabsf(v[j]));
  return top;
}
__device__ __forceinline__ int scale_exponent(const float (&v)[CB], float top) {
  if (!(top <= 3.4028235e38f)) {  // inf beside finite values: the scale is theirs
    top = 0.0f;
#pragma unroll
    for (int j = 0; j < CB; ++j)
      if (fabsf(v[j]) <= 3.4028235e38f) top = fmaxf(top, fabsf(v[j]));
  }
  // values below 2^(e + 1) times 2^(14 - e) stay below 2^15, inside fp16's range
  return max(-100, (int)(__float_as_uint(top) >> 23) - 127);
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

template <typename T>
__device__ __forceinline__ void save_gate_up(uint8_t* block, int lane, bool row_in, const float (&g)[CB], const float (&u)[CB]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *reinterpret_cast<float4*>(block + j * 512 + lane * 16) = make_float4(g[4 * j], g[4 * j + 1], g[4 * j + 2], g[4 * j + 3]);
      *reinterpret_cast<float4*>(block + 2048 + j * 512 + lane * 16) =
          make_float4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
    }
  } else {
    const float tg = largest(g), tu = largest(u);
    // a row past the matrix holds anything
    const bool fits = !row_in || (fminf(tg, tu) >= 0.0625f && fmaxf(tg, tu) < 32768.0f);
    int eg = 14, eu = 14;
    if (__all_sync(0xffffffffu, fits)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        *reinterpret_cast<uint4*>(block + j * 512 + lane * 16) = pack8<__half>(g, j);
        *reinterpret_cast<uint4*>(block + 1024 + j * 512 + lane * 16) = pack8<__half>(u, j);
      }
    } else {
      // per row: what a row keeps does not depend on its neighbours
      eg = fits ? 14 : scale_exponent(g, tg);
      eu = fits ? 14 : scale_exponent(u, tu);
      const float sg = exp2_int(14 - eg), su = exp2_int(14 - eu);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        *reinterpret_cast<uint4*>(block + j * 512 + lane * 16) = pack8<__half>(g, j, sg);
        *reinterpret_cast<uint4*>(block + 1024 + j * 512 + lane * 16) = pack8<__half>(u, j, su);
      }
    }
    reinterpret_cast<uint16_t*>(block + 2048)[lane] = (uint16_t)((eg & 0xff) | (eu & 0xff) << 8);
  }
}
// A lane's share of a saved block, fetched ahead of its use and then decoded.
template <typename T>
struct SavedRaw {
  static constexpr int kPieces = sizeof(T) == 4 ? 4 : 2;
  uint4 a[kPieces], b[kPieces];
  uint16_t e;
  __device__ __forceinline__ void load(const uint8_t* block, int lane) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      a[j] = *reinterpret_cast<const uint4*>(block + j * 512 + lane * 16);
      b[j] = *reinterpret_cast<const uint4*>(block + kPieces * 512 + j * 512 + lane * 16);
    }
    e = sizeof(T) == 4 ? 0 : reinterpret_cast<const uint16_t*>(block + 2048)[lane];
  }
  __device__ __forceinline__ void decode(float (&g)[CB], float (&u)[CB]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        g[4 * j] = __uint_as_float(a[j].x); g[4 * j + 1] = __uint_as_float(a[j].y);
        g[4 * j + 2] = __uint_as_float(a[j].z); g[4 * j + 3] = __uint_as_float(a[j].w);
        u[4 * j] = __uint_as_float(b[j].x); u[4 * j + 1] = __uint_as_float(b[j].y);
        u[4 * j + 2] = __uint_as_float(b[j].z); u[4 * j + 3] = __uint_as_float(b[j].w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t aw[4] = {a[j].x, a[j].y, a[j].z, a[j].w}, bw[4] = {b[j].x, b[j].y, b[j].z, b[j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&aw[k]));
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&bw[k]));
          g[8 * j + 2 * k] = x.x; g[8 * j + 2 * k + 1] = x.y;
          u[8 * j + 2 * k] = y.x; u[8 * j + 2 * k + 1] = y.y;
        }
      }
      if (!__all_sync(0xffffffffu, e == (14 | 14 << 8))) {
        // the exponents as signed bytes; -100 and up, so 2^(e - 14) is a normal number
        const float sg = exp2_int((int)(int8_t)(e & 0xff) - 14), su = exp2_int((int)(int8_t)(e >> 8) - 14);
#pragma unroll
        for (int j = 0; j < CB; ++j) {
          g[j] *= sg;
          u[j] *= su;
        }
      }
    }
  }
};

// ---------------------------------------------------------------- column sums of a block
// 16-bit data: a block of fp32 values, before their rounding (rounded ones
// would put as much error into a sum of mixed signs as the result's own
// rounding does), staged as [32 rows][16] with the 16-byte pieces of row r at
// j ^ (r / 2 % 4), so eight lanes cover all banks; lane l then adds piece l % 4
// of rows l / 4, l / 4 + 8, ...  (By mma.sync with a row operand of ones: 150
// us more in the 92416 x 2048 pass; the legacy instruction takes the tensor
// cores' time.)
__device__ __forceinline__ void staged_column_sums(uint8_t* rows, int lane, const float (&v)[CB], float (&sum)[4]) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < CB / 4; ++j)
    *reinterpret_cast<float4*>(rows + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
        make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (lane >> 2) + 8 * i;
    const float4 f = *reinterpret_cast<const float4*>(rows + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
    sum[0] += f.x; sum[1] += f.y; sum[2] += f.z; sum[3] += f.w;
  }
}
// The eight row groups (lane / 4) of two such blocks meet, each step halving
// what a lane holds: lane l returns block l / 16's column 4 (l % 4) + 2 (l / 8 %
// 2) + l / 4 % 2.
__device__ __forceinline__ float meet_row_groups(int lane, const float (&a)[4], const float (&b)[4]) {
  float s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float other = __shfl_xor_sync(0xffffffffu, lane & 16 ? a[j] : b[j], 16);
    s[j] = (lane & 16 ? b[j] : a[j]) + other;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float other = __shfl_xor_sync(0xffffffffu, lane & 8 ? s[j] : s[j + 2], 8);
    s[j] = (lane & 8 ? s[j + 2] : s[j]) + other;
  }
  const float other = __shfl_xor_sync(0xffffffffu, lane & 4 ? s[0] : s[1], 4);
  return (lane & 4 ? s[1] : s[0]) + other;
}
// fp32: lanes 0-15 return the sums of columns 0-15 over the warp's lanes, in an
// order fixed by the lanes.
__device__ __forceinline__ float column_sum(float (&v)[CB], int lane) {
#pragma unroll
  for (int j = 0; j < CB; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], 16);
#pragma unroll
  for (int half = 8; half; half >>= 1) {
    const bool up = (lane & half) != 0;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float keep = up ? v[j + half] : v[j];
      const float send = up ? v[j] : v[j + half];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, send, half);
    }
  }
  return v[0];
}

// ---------------------------------------------------------------- work
// The pieces of a worker: whole tiles worker, worker + workers, ..., then its
// share of the cut ones (struct Cut).  CUT: the product may have cut tiles (the
// gated passes never do, and keep the registers that this takes).
template <bool CUT>
struct Work {
  int worker, workers, nkb;
  int at, whole_end;            // whole tiles: at, at + workers, ... below whole_end
  int64_t unit, unit_end;       // units still to do of a run
  bool slice;                   // the slice is still to do
  int tile, kb0, kb1, slot;     // the current piece; slot < 0: a whole tile
  DCN_HOST_DEVICE Work(const GemmArgs& a, int worker_, int workers_)
      : worker(worker_), workers(workers_), nkb(a.nk * a.nseg), at(worker_), unit(0), unit_end(0), slice(false) {
    whole_end = a.tiles_m * a.tiles_n * a.batches;
    if (CUT && a.split) {
      whole_end -= a.cut.R;
      const int e = worker - a.cut.S * a.cut.R;
      slice = e < 0;
      if (!slice && e < a.cut.E) {
        unit = a.cut.units() * e / a.cut.E;
        unit_end = a.cut.units() * (e + 1) / a.cut.E;
      }
    }
  }
  DCN_HOST_DEVICE bool next(const GemmArgs& a) {
    if (at < whole_end) {
      tile = at;
      at += workers;
      kb0 = 0;
      kb1 = nkb;
      slot = -1;
      return true;
    }
    if (!CUT) return false;
    const Cut& c = a.cut;
    if (slice) {
      slice = false;
      const int s = worker / c.R;
      tile = whole_end + worker - s * c.R;
      kb0 = s * c.a;
      kb1 = min(nkb, kb0 + c.a);
      slot = worker;
      return true;
    }
    if (unit >= unit_end) return false;
    const int t = (int)(unit / c.rest);
    const int k = (int)(unit - (int64_t)t * c.rest);
    const int len = (int)min((int64_t)(c.rest - k), unit_end - unit);
    tile = whole_end + t;
    kb0 = c.S * c.a + k;
    kb1 = kb0 + len;
    slot = worker + t;
    unit += len;
    return true;
  }
};

// Tile index -> (batch, row tile, column tile): blocks of kGroupM row tiles,
// row tiles fastest inside a block, so the CTAs of a wave share both operands
// in the L2.
__host__ __device__ __forceinline__ void tile_at(const GemmArgs& a, int tile, int& z, int& mt, int& nt) {
  z = (int)a.per_batch((uint32_t)tile);
  int t = tile - z * (a.tiles_m * a.tiles_n);
  const int block = (int)a.per_block((uint32_t)t);
  t -= block * (kGroupM * a.tiles_n);
  const bool last = (block + 1) * kGroupM > a.tiles_m;
  nt = last ? (int)a.last_rows((uint32_t)t) : t / kGroupM;
  mt = block * kGroupM + t - nt * (last ? a.tiles_m - block * kGroupM : kGroupM);
}
inline void set_tiles(GemmArgs& a, int tiles_m, int tiles_n, int batches) {
  a.tiles_m = tiles_m;
  a.tiles_n = tiles_n;
  a.batches = batches;
  a.per_batch = fast_div((uint32_t)(tiles_m * tiles_n));
  a.per_block = fast_div((uint32_t)(kGroupM * tiles_n));
  a.last_rows = fast_div((uint32_t)(tiles_m % kGroupM ? tiles_m % kGroupM : kGroupM));
}

// ---------------------------------------------------------------- kernel
// A, B: the operand's form.
enum Form { ROWS_K, ROWS_MN, PANELS_K, PANELS_MN };

template <typename T, int EPI, int BN, Form A, Form B, bool PAIR>
__global__ void __launch_bounds__(NTHREADS, 1)
ffn_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ GemmArgs a) {
  constexpr bool A_MN = A == ROWS_MN || A == PANELS_MN, B_MN = B == ROWS_MN || B == PANELS_MN;
  constexpr int S = stages(EPI, BN, PAIR, sizeof(T) == 4);
  constexpr uint32_t STAGING = staging_bytes(EPI, BN, sizeof(T) == 4);  // of a warp
  constexpr uint32_t STAGE = stage_bytes(BN, PAIR);
  constexpr bool GATED = EPI == EPI_GATED, RECOMP = EPI == EPI_RECOMPUTE, TWO = GATED || RECOMP;
  constexpr bool DGATE = EPI == EPI_DGATE || RECOMP;
  constexpr int COLS = GATED ? BN / 2 : RECOMP ? BN / 3 : BN;  // output columns of a tile
  constexpr int ACC = RECOMP ? 256 : BN;                       // TMEM columns of an accumulator buffer
  constexpr uint32_t B_AT = (RECOMP ? 2 : 1) * A_STAGE;        // column operands in a stage
  constexpr int CTAS = PAIR ? 2 : 1;
  constexpr bool WIDE = sizeof(T) == 4;
  // K blocks of one accumulation in TMEM.  The tensor cores truncate each
  // addition to the accumulator, an error that grows with the number of steps
  // (measured on fp32 data: 2.4e-6 of the result's norm after 128 steps, where
  // sums rounded to nearest leave 6e-7); fp32 data therefore moves its sums to
  // registers every kWideRun blocks.  16-bit results do not see the difference.
  constexpr int RUN = WIDE ? kWideRun : 1 << 30;
  static_assert(!WIDE || BN <= 128 || RECOMP, "an epilogue thread holds 32 to 48 sums");
  static_assert(RECOMP == (BN == kRecomputeBn), "accumulator columns");
  static_assert(!PAIR || !RECOMP, "half of 64 dhidden columns fills no swizzled row");
  constexpr int STEP = EPI_WARPS / 4;  // warps that share 32 rows of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_addr(smem);
  uint8_t* staging = smem + S * STAGE;
  uint8_t* tail = staging + EPI_WARPS * STAGING + kBiasBytes;
  if (smem - smem_raw > kSmemSlack) {  // an unexpected start (the same in both CTAs): nothing is touched
    if (threadIdx.x == 0) atomicExch(a.status, ST_FFN_SMEM);
    return;
  }
  const uint32_t bar0 = smem_addr(tail);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (S + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * S + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * S + 2 + b); };
  const uint32_t drain = bar0 + 8u * (2 * S + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + (2 * S + 5) * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + (2 * S + 5) * 8 + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_rank() : 0;
  constexpr uint32_t TMEM_COLS = 2 * ACC;
  constexpr bool FREE = !PAIR && (GATED || (EPI == EPI_STORE && B == ROWS_K));
  const int cols = FREE ? a.cols : COLS;
  const uint32_t tx = FREE ? a.a_bytes + (uint32_t)cols * (GATED ? 256u : 128u) : (uint32_t)CTAS * STAGE;  // of a stage

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), EPI_WARPS * CTAS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == MMA_WARP) tmem_alloc_g<PAIR>(smem_addr(tmem_slot), TMEM_COLS);
  tc_fence_before();
  if (PAIR) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Work<EPI == EPI_STORE> w(a, blockIdx.x / CTAS, gridDim.x / CTAS);

  if (warp >= EPI_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == LOAD_WARP) {
      // ------------------------------------------------ TMA loads
      if (lane == 0) {
        int issued = 0;
        bool ok = true;
        while (ok && w.next(a)) {
          int z, mt, nt;
          tile_at(a, w.tile, z, mt, nt);
          const int m0 = (mt * CTAS + rank) * BM, n0 = nt * cols;
          const int nb = PAIR && !GATED ? n0 + rank * (BN / 2) : n0;  // this CTA's part of the column operand
          int sg = w.kb0 / a.nk, kb = w.kb0 - sg * a.nk;
          for (int i = w.kb0; i < w.kb1; ++i) {
            const int s = issued % S;
            ok = mbar_wait(empty(s), ((issued / S) & 1) ^ 1, abort_flag, a.status, ST_FFN_LOAD);
            if (!ok) break;
            const Seg seg = a.seg[sg];
            const int k = kb * BK;
            const uint32_t dst = sbase + s * STAGE;
            const uint32_t bar = PAIR ? in_first_cta(full(s)) : full(s);
            const CUtensorMap* ma = &maps.m[seg.a_map + z];
            const CUtensorMap* mb = &maps.m[seg.b_map];
            if (rank == 0) mbar_arrive_expect_tx(full(s), tx);
            if (A == PANELS_MN) {
              load_panels<PAIR>(dst, ma, k, m0 >> 3, seg.a_plane, bar);
            } else if (A == PANELS_K) {
              load_panels<PAIR>(dst, ma, m0, k >> 3, seg.a_plane, bar);
            } else if (A == ROWS_MN) {
              load_g<PAIR>(dst, ma, m0, k, seg.a_plane, bar);
              load_g<PAIR>(dst + 8192, ma, m0 + 64, k, seg.a_plane, bar);
            } else {
              load_g<PAIR>(dst, ma, k, m0, seg.a_plane, bar);
            }
            if (GATED && PAIR) {
              load_g<PAIR>(dst + B_AT, mb + rank, k, n0, seg.b_plane, bar);
            } else if (TWO) {
              tma_load_3d(dst + B_AT, mb, k, n0, seg.b_plane, bar);
              tma_load_3d(dst + B_AT + cols * 128, mb + 1, k, n0, seg.b_plane, bar);
              if (RECOMP) {  // dy beside x, w_down (MN-major) beside the other two
                tma_load_3d(dst + A_STAGE, ma + 1, k, m0, seg.a_plane, bar);
                tma_load_3d(dst + B_AT + 2 * COLS * 128, mb + 2, n0, k, seg.b_plane, bar);
              }
            } else if (B == PANELS_MN) {
              load_panels<PAIR>(dst + A_STAGE, mb, k, nb >> 3, seg.b_plane, bar);
            } else if (B == ROWS_MN) {
#pragma unroll
              for (int q = 0; q < BN / 64 / CTAS; ++q)
                load_g<PAIR>(dst + A_STAGE + q * 8192, mb, nb + 64 * q, k, seg.b_plane, bar);
            } else {
              load_g<PAIR>(dst + A_STAGE, mb, k, nb, seg.b_plane, bar);
            }
            ++issued;
            if (++kb == a.nk) {
              kb = 0;
              ++sg;
            }
          }
        }
        // copies in flight land before the CTA may go (a pair's report to the first CTA)
        if (rank == 0)
          for (int i = issued > S ? issued - S : 0; i < issued; ++i)
            mbar_wait(full(i % S), (i / S) & 1, abort_flag, a.status, ST_FFN_DRAIN);
      }
    } else if (warp == MMA_WARP) {
      // ------------------------------------------------ MMA issuer
      if (lane == 0 && rank == 0) {
        const uint32_t idesc = tcc::idesc_f16_major(BM * CTAS, TWO ? 2 * cols : FREE ? cols : BN, a.operand_bf16 != 0, A_MN, B_MN);
        const uint32_t idesc_dh = tcc::idesc_f16_major(BM, COLS, a.operand_bf16 != 0, false, true);
        int used = 0, done = 0;
        bool ok = true;
        while (ok && w.next(a)) {
          for (int k0 = w.kb0; ok && k0 < w.kb1; k0 += RUN) {
            const int k1 = w.kb1 - k0 > RUN ? k0 + RUN : w.kb1;
            const int b = done & 1;
            ok = mbar_wait(acc_empty(b), ((done >> 1) & 1) ^ 1, abort_flag, a.status, ST_FFN_MMA);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(b * ACC);
            for (int i = k0; i < k1; ++i) {
              const int s = used % S;
              ok = mbar_wait(full(s), (used / S) & 1, abort_flag, a.status, ST_FFN_MMA);
              if (!ok) break;
              tc_fence_after();
              const uint32_t ab = sbase + s * STAGE, bb = ab + B_AT;
#pragma unroll
              for (int kk = 0; kk < BK / 16; ++kk) {
                // panels in shared memory: K-major [panel][128 rows][16 B] (panels along K by
                // LBO, 8-row groups by SBO); MN-major [panel][64 rows][16 B] (8-row groups along
                // K by LBO, panels by SBO)
                const uint64_t ad = A == PANELS_K    ? (FREE ? desc_panels(ab + kk * 2 * a.a_lbo, a.a_lbo, 128) : desc_panels(ab + kk * 4096, 2048, 128))
                                    : A == PANELS_MN ? desc_panels(ab + kk * 256, 128, 1024)
                                    : A == ROWS_MN   ? tcc::desc_mnmajor_sw128(ab + kk * 2048, 8192)
                                                     : desc_kmajor_sw128(ab + kk * 32);
                const uint64_t bd = B == PANELS_MN ? desc_panels(bb + kk * 256, 128, 1024)
                                    : B == ROWS_MN ? tcc::desc_mnmajor_sw128(bb + kk * 2048, 8192)
                                                   : desc_kmajor_sw128(bb + kk * 32);
                mma_g<PAIR>(d, ad, bd, idesc, (i > k0 || kk > 0) ? 1u : 0u);
                if (RECOMP)
                  mma_f16(d + 2 * COLS, desc_kmajor_sw128(ab + A_STAGE + kk * 32),
                          tcc::desc_mnmajor_sw128(bb + 2 * COLS * 128 + kk * 2048, 8192), idesc_dh,
                          (i > k0 || kk > 0) ? 1u : 0u);
              }
              commit_g<PAIR>(empty(s), true);
              ++used;
            }
            if (!ok) break;
            commit_g<PAIR>(acc_full(b), true);
            ++done;
          }
        }
        // MMAs still running finish before TMEM and shared memory are released
        if (used > 0) {
          commit_g<PAIR>(drain, false);
          mbar_wait(drain, 0, abort_flag, a.status, ST_FFN_DRAIN);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    // ------------------------------------------------ epilogue
    const int q = warp & 3;  // lanes 32 q ..
    // of the tile's column blocks: STORE a run of its own, else first, first + STEP, ...
    constexpr int BLOCKS = COLS / CB;
    constexpr bool RUNS = EPI == EPI_STORE && !WIDE;
    constexpr int MINE = BLOCKS / STEP > 0 ? BLOCKS / STEP : 1;  // blocks of a warp (BLOCKS = 2: of two warps in four)
    const int first = RUNS ? (warp >> 2) * MINE : warp >> 2;
    constexpr int NEXT = RUNS ? 1 : STEP;
    const int end = RUNS ? min(first + MINE, cols / CB) : cols / CB;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    uint8_t* stage = staging + warp * STAGING;
    float* colf = reinterpret_cast<float*>(staging + EPI_WARPS * STAGING) + warp * 32;
    const bool has_bias = EPI != EPI_DGATE && a.bias[0] != nullptr;
    const int64_t col_blocks = (a.N + CB - 1) / CB;
    // The bias values of a block, one a lane (RECOMPUTE, GATED: 16 of gate, 16
    // of up), fetched ahead and read back by all lanes through the warp's own
    // piece of shared memory.
    auto bias_of = [&](int c0) {
      const int k = lane >> 4, c = c0 + (lane & 15);
      return (k == 0 || TWO) && c < a.N ? static_cast<const T*>(a.bias[k])[c] : from_f<T>(0.0f);
    };
    int done = 0;
    bool ok = true;
    auto wait_acc = [&] {
      ok = mbar_wait(acc_full(done & 1), (done >> 1) & 1, abort_flag, a.status, ST_FFN_EPI);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) tc_fence_after();
      return ok;
    };
    auto release_acc = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(in_first_cta(acc_empty(done & 1)));
        else mbar_arrive_relaxed(acc_empty(done & 1));
      }
      ++done;
    };
    while (ok && w.next(a)) {
      int z, mt, nt;
      tile_at(a, w.tile, z, mt, nt);
      const int n0 = nt * cols;
      const int row0 = (mt * CTAS + rank) * BM + q * 32;
      const int64_t row = (int64_t)row0 + lane;
      const bool row_in = row < a.M;
      const bool whole = w.slot < 0;
      const int64_t m_block = row0 / 32;
      auto saved_block = [&](int c) {
        return static_cast<uint8_t*>(a.saved) + saved_block_offset<T>(m_block, n0 / CB + c, col_blocks);
      };

      // One block of this tile.  v: its sums (GATED, RECOMPUTE: gate); u: up (from
      // TMEM or, DGATE, the saved state with gate in v's place); dh: dhidden.
      auto block = [&](int c, float (&v)[CB], float (&u)[CB], float (&dh)[CB], T bias) {
        const int c0 = n0 + c * CB;
        if (!whole) {
          if (row0 >= a.M) return;
          // an fp32 partial of this tile, 16-byte pieces of 32 rows side by side
          float* slot = a.partial + ((int64_t)w.slot * CTAS + rank) * (BM * BN) + q * (32 * BN);
#pragma unroll
          for (int j = 0; j < CB / 4; ++j)
            *reinterpret_cast<float4*>(slot + c * 512 + j * 128 + lane * 4) =
                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          return;
        }
        if (c0 >= a.N) return;
        if (has_bias) {
          __syncwarp();
          colf[lane] = to_f<T>(bias);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < CB / 4; ++j) {
            const float4 f = reinterpret_cast<const float4*>(colf)[j];
            v[4 * j] += f.x; v[4 * j + 1] += f.y; v[4 * j + 2] += f.z; v[4 * j + 3] += f.w;
            if (TWO) {
              const float4 h = reinterpret_cast<const float4*>(colf + CB)[j];
              u[4 * j] += h.x; u[4 * j + 1] += h.y; u[4 * j + 2] += h.z; u[4 * j + 3] += h.w;
            }
          }
        }
        // this row in the panels of the block's columns; rows past M are zero
        // there, to the end of their 128
        const bool rows_in = row0 - q * 32 < a.M;
        const int64_t at = ((int64_t)(row0 >> 7) * a.ldo + (c0 >> 3)) * (BM * 16) + (q * 32 + lane) * 16;
        if constexpr (GATED) {
          if (a.saved) save_gate_up<T>(saved_block(c), lane, row_in, v, u);
          gate_block<WIDE>(a.act, v, u, v);
          if (row0 + 32 > a.M && !row_in) {
#pragma unroll
            for (int j = 0; j < CB; ++j) v[j] = 0.0f;
          }
          if (rows_in) store_panels<T>(static_cast<uint8_t*>(a.out[0]) + at, a.plane, a.N - c0, v);
        } else if constexpr (DGATE) {
          dgate_block<WIDE>(a.act, dh, v, u);
          if (row0 + 32 > a.M && !row_in) {
#pragma unroll
            for (int j = 0; j < CB; ++j) v[j] = u[j] = 0.0f;
          }
          if (rows_in) {
            store_panels<T>(static_cast<uint8_t*>(a.out[0]) + at, a.plane, a.N - c0, v);
            store_panels<T>(static_cast<uint8_t*>(a.out[1]) + at, a.plane, a.N - c0, u);
          }
          if (a.colsum) {
            float* sums = a.colsum + (m_block * 2) * a.N;
            if constexpr (WIDE) {
              const float sg = column_sum(v, lane), su = column_sum(u, lane);
              if (lane < CB && c0 + lane < a.N) {
                sums[c0 + lane] = sg;
                sums[a.N + c0 + lane] = su;
              }
            } else {
              float sg[4], su[4];
              staged_column_sums(stage, lane, v, sg);
              staged_column_sums(stage, lane, u, su);
              const float sum = meet_row_groups(lane, sg, su);
              const int c = c0 + 4 * (lane & 3) + 2 * (lane >> 3 & 1) + (lane >> 2 & 1);
              if (c < a.N) sums[(lane >> 4) * a.N + c] = sum;
            }
          }
        } else {
          if (!WIDE && a.vec) {
            if constexpr (!WIDE) {
              // the last tile's store has read the staged rows
              if (c == first) {
                if (lane == 0) bulk_wait_read_all();
                __syncwarp();
              }
              stage_row<T, BN / 2>(stage, lane, c - first, v);
            }
          } else if (row_in) {
            store_row<T>(static_cast<T*>(a.out[z]) + row * a.ldo, c0, a.N, a.vec != 0, v);
          }
        }
      };

      // what the first block needs from memory is fetched while the products
      // run, the next ones' a block ahead
      const bool use_bias = has_bias && whole;
      T bias = from_f<T>(0.0f);
      if (use_bias) bias = bias_of(n0 + first * CB);
      SavedRaw<T> raw;
      if (EPI == EPI_DGATE && first < end && n0 + first * CB < a.N) raw.load(saved_block(first), lane);
      if constexpr (WIDE) {
        // this thread's sums, added up over the runs: at most two blocks
        constexpr int NB = BLOCKS > 4 ? 2 : 1;
        static_assert(BLOCKS <= 8, "blocks of a warp");
        float sum[NB][CB], sum_u[TWO ? NB : 1][CB], sum_dh[RECOMP ? NB : 1][CB];
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int j = 0; j < CB; ++j) {
            sum[k][j] = 0.0f;
            if (TWO) sum_u[k][j] = 0.0f;
            if (RECOMP) sum_dh[k][j] = 0.0f;
          }
        for (int k0 = w.kb0; k0 < w.kb1; k0 += RUN) {
          if (!wait_acc()) break;
          const uint32_t acc = lanes + (uint32_t)((done & 1) * ACC);
#pragma unroll
          for (int k = 0; k < NB; ++k) {
            const int c = first + STEP * k;
            if (c >= end) break;
            float t[CB];
            tmem_load(acc + c * CB, t);
            tmem_wait(t);
#pragma unroll
            for (int j = 0; j < CB; ++j) sum[k][j] += t[j];
            if constexpr (TWO) {
              tmem_load(acc + cols + c * CB, t);
              tmem_wait(t);
#pragma unroll
              for (int j = 0; j < CB; ++j) sum_u[k][j] += t[j];
            }
            if constexpr (RECOMP) {
              tmem_load(acc + 2 * COLS + c * CB, t);
              tmem_wait(t);
#pragma unroll
              for (int j = 0; j < CB; ++j) sum_dh[k][j] += t[j];
            }
          }
          release_acc();
        }
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const int c = first + STEP * k;
          if (c >= end) break;
          if (k > 0 && use_bias) bias = bias_of(n0 + c * CB);
          if constexpr (EPI == EPI_DGATE) {
            if (k > 0 && n0 + c * CB < a.N) raw.load(saved_block(c), lane);
            float g[CB], u[CB];
            raw.decode(g, u);
            block(c, g, u, sum[k], bias);
          } else {
            block(c, sum[k], sum_u[TWO ? k : 0], sum_dh[RECOMP ? k : 0], bias);
          }
        }
      } else {
        if (!wait_acc()) break;
        const uint32_t acc = lanes + (uint32_t)((done & 1) * ACC);
        // v: gate or plain sums or (DGATE) dhidden; u: up; dh: RECOMPUTE's dhidden
        auto read = [&](int c, float (&v)[CB], float (&u)[CB], float (&dh)[CB]) {
          tmem_load(acc + c * CB, v);
          if (TWO) tmem_load(acc + cols + c * CB, u);
          if (RECOMP) tmem_load(acc + 2 * COLS + c * CB, dh);
          tmem_wait(v);
          if (TWO) tmem_wait(u);
          if (RECOMP) tmem_wait(dh);
        };
        float v[CB], u[CB], dh[CB];
        if (first < end) read(first, v, u, dh);
        if (first + NEXT >= end) release_acc();
#pragma unroll 1
        for (int c = first; c < end; c += NEXT) {
          const bool more = c + NEXT < end;
          const T now = bias;
          float nv[CB], nu[CB], ndh[CB];
          if (more) {
            read(c + NEXT, nv, nu, ndh);
            if (c + 2 * NEXT >= end) release_acc();
          }
          const bool inside = more && n0 + (c + NEXT) * CB < a.N;
          if (inside && use_bias) bias = bias_of(n0 + (c + NEXT) * CB);
          if constexpr (EPI == EPI_DGATE) {
            float g[CB], up[CB];
            raw.decode(g, up);
            if (inside) raw.load(saved_block(c + NEXT), lane);
            block(c, g, up, v, now);
          } else {
            block(c, v, u, dh, now);
          }
#pragma unroll
          for (int j = 0; j < CB; ++j) {
            v[j] = nv[j];
            if (TWO) u[j] = nu[j];
            if (RECOMP) dh[j] = ndh[j];
          }
        }
        if constexpr (RUNS) {
          // the staged columns leave; the writes reach the TMA first
          if (whole && a.vec && n0 + first * CB < a.N) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0 && row0 < a.M) {
              tma_store_3d(&maps.out[z], smem_addr(stage), n0 + first * CB, row0, 0);
              bulk_commit();
            }
          }
        }
      }
    }
    // the stores have left shared memory and are done before the CTA ends
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  if (PAIR) cluster_sync();  // neither CTA's memory is in use by the other any more
  else __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc_g<PAIR>(tmem, TMEM_COLS);
  }
  if (PAIR) cluster_sync();
}

}  // namespace ffn
}  // namespace dcn
