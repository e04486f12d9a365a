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
// Warp roles (320 threads): warps 0-7 epilogue, warp 8 issues the MMAs, warp 9
// the TMA loads.  A CTA works through its share of the output tiles; the
// accumulator is double-buffered in TMEM (2 x BN columns), so a tile's
// epilogue runs under the next tile's MMAs.  Epilogue warp w reads TMEM lanes
// 32 (w % 4) .. +31: lane i owns one row, 32 columns at a time.
//
// Work is dealt in whole tiles: worker w takes tiles w, w + W, ...  Where the
// last wave would leave many of the W workers idle, its R tiles are cut along
// K instead (struct Cut): S = W / R workers a tile walk S equal slices of K,
// tile by tile side by side, so that at any time all tiles read the same rows
// of both operands and these come from the L2 (dealt tile after tile, a
// product with a long K reads them from memory once per tile); the W - S R
// workers left over share the end of K in equal runs.  Each piece is an fp32
// partial in a slot of its own, and a second kernel adds a tile's slots in a
// fixed order: the result does not depend on timing.
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

constexpr int EPI_WARPS = 8;
constexpr int MMA_WARP = 8, LOAD_WARP = 9;
constexpr int NTHREADS = 320;
constexpr uint32_t A_STAGE = BM * 128;
constexpr int ST_FFN_LOAD = 61, ST_FFN_MMA = 62, ST_FFN_EPI = 63, ST_FFN_DRAIN = 64, ST_FFN_SMEM = 65;

__host__ __device__ constexpr int stages(int bn) { return bn == 256 ? 4 : bn == 128 ? 6 : 8; }
__host__ __device__ constexpr uint32_t stage_bytes(int bn) { return A_STAGE + (uint32_t)bn * 128u; }
// operand stages, then two staged output blocks and 64 bias values of each
// epilogue warp, then barriers
constexpr uint32_t kStaging = EPI_WARPS * 2 * 32 * 64;
__host__ __device__ constexpr uint32_t smem_bytes(int bn) {
  return (uint32_t)stages(bn) * stage_bytes(bn) + kStaging + EPI_WARPS * 64 * 4u +
         (2u * (uint32_t)stages(bn) + 5u) * 8u + 16u;
}
// dynamic shared memory starts on 1024 bytes when a kernel has no static one;
// this much is left over for a start that does not (checked by the kernel)
constexpr uint32_t kSmemSlack = 768;
static_assert(smem_bytes(256) + kSmemSlack <= 232448, "shared memory of one CTA");
// fp32 data: K blocks added up in TMEM before their sum moves on to registers
constexpr int kWideRun = 4;

enum Epi { EPI_GATED, EPI_DGATE, EPI_STORE };

struct Seg {
  uint8_t a_map, a_plane, b_map, b_plane;
};
struct Maps {
  CUtensorMap m[4];
  CUtensorMap out[2];  // 16-bit results, 32 x 32 blocks
};

struct GemmArgs {
  int M, N;                  // output extents (GATED, DGATE: N = F)
  int nk, nseg;              // K blocks of a segment, segments
  Seg seg[12];
  int tiles_m, tiles_n, batches;  // a batch adds its index to a_map (and picks the output)
  int group_m;               // tiles are dealt in blocks of group_m row tiles x all column tiles
  int split;                 // 1: the last tiles are cut along K (Cut), partials to `partial`
  int act;
  uint32_t operand_bf16;
  float* partial;
  // outputs: STORE: out[batch] [M][ldo] of T (+ bias); GATED: hidden; DGATE: dgate, dup.
  void* out[2];
  int64_t ldo;
  int64_t plane;             // fp32: elements between the bf16 planes of hidden / dgate / dup
  int vec;                   // out rows take 16-byte stores (16-bit data: TMA stores)
  const void* bias[2];       // STORE: [0]; GATED: gate, up
  // saved gate and up (private layout, below), and the hidden values' other copy
  void* saved;
  float* colsum;             // DGATE: [32-row block][2][F] column sums of dgate and dup, or null
  int* status;
};

// ---------------------------------------------------------------- saved gate / up
// What the backward needs of a 32-row x 32-column block (its rows being the
// lanes of one warp) lies together, each 16-byte piece of the 32 lanes side by
// side, so both passes move whole lines:
//   16-bit data: gate, up as fp16 times a power of two per (row, 32 columns)
//     that puts the row's largest value near fp16's upper end: 11 bits, not
//     bf16's 8, of values that the derivative multiplies, at the same size;
//     then one int16 per lane with the two exponents;
//   fp32 data: gate, up as fp32.
template <typename T>
struct SavedBlock {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr size_t kGate = kWide ? 4096 : 2048;                     // bytes of one of the two
  static constexpr size_t kBytes = saved_block_bytes(kWide);
};
template <typename T>
__host__ __device__ inline size_t saved_block_offset(int64_t m_block, int64_t col_block, int64_t col_blocks) {
  return (size_t)(m_block * col_blocks + col_block) * SavedBlock<T>::kBytes;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Waits for this warp's TMEM loads; the values pass through, so that nothing
// that uses them is scheduled before the wait.
__device__ __forceinline__ void tmem_ld32_wait(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
      "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
      "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
      "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
      "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
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

// ---------------------------------------------------------------- activations
// ACCURATE (fp32 data): CUDA's expf and IEEE division; else the fast forms,
// whose few ulp are far below a 16-bit result's rounding.
template <bool ACCURATE>
__device__ __forceinline__ float sigmoid(float x) {
  // for x below -88 the exponential overflows to inf and the quotient is 0, as it should be
  return ACCURATE ? 1.0f / (1.0f + expf(-x)) : __fdividef(1.0f, 1.0f + __expf(-x));
}
template <bool ACCURATE, int ACT>
__device__ __forceinline__ float act_value(float x) {
  if constexpr (ACT == kActSilu) return x * sigmoid<ACCURATE>(x);
  else if constexpr (ACT == kActGelu) return x * (0.5f * (1.0f + erff(x * 0.70710678118654752f)));
  else if constexpr (ACT == kActRelu) return x > 0.0f ? x : (x == x ? 0.0f : x);
  else return sigmoid<ACCURATE>(x);
}
// act(x) and act'(x)
template <bool ACCURATE, int ACT>
__device__ __forceinline__ float2 act_both(float x) {
  if constexpr (ACT == kActSilu) {
    const float s = sigmoid<ACCURATE>(x);
    return make_float2(x * s, s * (1.0f + x * (1.0f - s)));
  } else if constexpr (ACT == kActGelu) {
    const float c = 0.5f * (1.0f + erff(x * 0.70710678118654752f));
    const float e = ACCURATE ? expf(-0.5f * x * x) : __expf(-0.5f * x * x);
    return make_float2(x * c, c + x * (0.39894228040143268f * e));
  } else if constexpr (ACT == kActRelu) {
    return x > 0.0f ? make_float2(x, 1.0f) : make_float2(x == x ? 0.0f : x, 0.0f);
  } else {
    const float s = sigmoid<ACCURATE>(x);
    return make_float2(s, s * (1.0f - s));
  }
}
// A row's 32 columns at a time; the activation is picked once for all of them.
template <bool ACCURATE, int ACT>
__device__ __forceinline__ void gate32(const float (&g)[32], const float (&u)[32], float (&h)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) h[j] = act_value<ACCURATE, ACT>(g[j]) * u[j];
}
// (gate, up) to (dgate, dup)
template <bool ACCURATE, int ACT>
__device__ __forceinline__ void dgate32(const float (&dh)[32], float (&g)[32], float (&u)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float2 s = act_both<ACCURATE, ACT>(g[j]);
    g[j] = dh[j] * u[j] * s.y;
    u[j] = dh[j] * s.x;
  }
}
template <bool ACCURATE>
__device__ __forceinline__ void gate32(int act, const float (&g)[32], const float (&u)[32], float (&h)[32]) {
  if (act == kActSilu) gate32<ACCURATE, kActSilu>(g, u, h);
  else if (act == kActGelu) gate32<ACCURATE, kActGelu>(g, u, h);
  else if (act == kActRelu) gate32<ACCURATE, kActRelu>(g, u, h);
  else gate32<ACCURATE, kActSigmoid>(g, u, h);
}
template <bool ACCURATE>
__device__ __forceinline__ void dgate32(int act, const float (&dh)[32], float (&g)[32], float (&u)[32]) {
  if (act == kActSilu) dgate32<ACCURATE, kActSilu>(dh, g, u);
  else if (act == kActGelu) dgate32<ACCURATE, kActGelu>(dh, g, u);
  else if (act == kActRelu) dgate32<ACCURATE, kActRelu>(dh, g, u);
  else dgate32<ACCURATE, kActSigmoid>(dh, g, u);
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

// 32 columns of one row of a row-major matrix of T with `n` columns.
template <typename T>
__device__ __forceinline__ void store_row32(T* row, int c0, int n, bool vec, const float (&v)[32]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + 4 * j < n)
          *reinterpret_cast<float4*>(row + c0 + 4 * j) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + 8 * j < n) {
          uint4 p;
          p.x = pack2(v[8 * j], v[8 * j + 1], (T*)nullptr);
          p.y = pack2(v[8 * j + 2], v[8 * j + 3], (T*)nullptr);
          p.z = pack2(v[8 * j + 4], v[8 * j + 5], (T*)nullptr);
          p.w = pack2(v[8 * j + 6], v[8 * j + 7], (T*)nullptr);
          *reinterpret_cast<uint4*>(row + c0 + 8 * j) = p;
        }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c0 + j < n) row[c0 + j] = from_f<T>(v[j]);
  }
}

// A 32 x 32 block of 16-bit values leaves through shared memory and one TMA
// store per warp, whole 64-byte row pieces at a time (row-owning lanes would
// write 16 bytes to 32 different lines an instruction).  Staged rows are 64
// bytes with the 64-byte swizzle: 16-byte piece j of row r at j ^ (r / 2 % 4),
// so eight lanes cover all banks.  Rows and columns past the matrix are
// dropped by the store.
constexpr uint32_t kStageBlock = 32 * 64;
template <typename T>
__device__ __forceinline__ void stage_row32(uint8_t* block, int lane, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 p;
    p.x = pack2(v[8 * j], v[8 * j + 1], (T*)nullptr);
    p.y = pack2(v[8 * j + 2], v[8 * j + 3], (T*)nullptr);
    p.z = pack2(v[8 * j + 4], v[8 * j + 5], (T*)nullptr);
    p.w = pack2(v[8 * j + 6], v[8 * j + 7], (T*)nullptr);
    *reinterpret_cast<uint4*>(block + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = p;
  }
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(z), "r"(src)
               : "memory");
}

// 32 columns of one row of an operand of a following product: T itself, or
// for fp32 data three bf16 planes.  Rows are padded to 16 bytes (`ld`).
template <typename T>
__device__ __forceinline__ void store_operand32(void* base, int64_t plane, int64_t row, int64_t ld, int c0,
                                                const float (&v)[32]) {
  if constexpr (sizeof(T) == 4) {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(base) + row * ld;
    float r[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = v[j];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      store_row32<__nv_bfloat16>(p + k * plane, c0, (int)ld, true, r);
      // a plane that holds inf or NaN ends the expansion: the others are zero
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float hi = __bfloat162float(__float2bfloat16_rn(r[j]));
        r[j] = fabsf(hi) <= 3.4e38f ? r[j] - hi : 0.0f;
      }
    }
  } else {
    store_row32<T>(static_cast<T*>(base) + row * ld, c0, (int)ld, true, v);
  }
}

// ---------------------------------------------------------------- saved values
__device__ __forceinline__ int scale_exponent(const float (&v)[32]) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 32; ++j) top = fmaxf(top, fabsf(v[j]));
  if (!(top <= 3.4028235e38f)) {  // inf beside finite values: the scale is theirs
    top = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (fabsf(v[j]) <= 3.4028235e38f) top = fmaxf(top, fabsf(v[j]));
  }
  // values below 2^(e + 1) times 2^(14 - e) stay below 2^15, inside fp16's range
  return max(-100, (int)(__float_as_uint(top) >> 23) - 127);
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

template <typename T>
__device__ __forceinline__ void save_gate_up(uint8_t* block, int lane, const float (&g)[32], const float (&u)[32]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      *reinterpret_cast<float4*>(block + j * 512 + lane * 16) = make_float4(g[4 * j], g[4 * j + 1], g[4 * j + 2], g[4 * j + 3]);
      *reinterpret_cast<float4*>(block + 4096 + j * 512 + lane * 16) =
          make_float4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
    }
  } else {
    const int eg = scale_exponent(g), eu = scale_exponent(u);
    const float sg = exp2_int(14 - eg), su = exp2_int(14 - eu);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 a, b;
      a.x = pack2(g[8 * j] * sg, g[8 * j + 1] * sg, (__half*)nullptr);
      a.y = pack2(g[8 * j + 2] * sg, g[8 * j + 3] * sg, (__half*)nullptr);
      a.z = pack2(g[8 * j + 4] * sg, g[8 * j + 5] * sg, (__half*)nullptr);
      a.w = pack2(g[8 * j + 6] * sg, g[8 * j + 7] * sg, (__half*)nullptr);
      b.x = pack2(u[8 * j] * su, u[8 * j + 1] * su, (__half*)nullptr);
      b.y = pack2(u[8 * j + 2] * su, u[8 * j + 3] * su, (__half*)nullptr);
      b.z = pack2(u[8 * j + 4] * su, u[8 * j + 5] * su, (__half*)nullptr);
      b.w = pack2(u[8 * j + 6] * su, u[8 * j + 7] * su, (__half*)nullptr);
      *reinterpret_cast<uint4*>(block + j * 512 + lane * 16) = a;
      *reinterpret_cast<uint4*>(block + 2048 + j * 512 + lane * 16) = b;
    }
    reinterpret_cast<uint16_t*>(block + 4096)[lane] = (uint16_t)((eg & 0xff) | (eu & 0xff) << 8);
  }
}
// A lane's share of a saved block, fetched ahead of its use and then decoded.
template <typename T>
struct SavedRaw {
  static constexpr int kPieces = sizeof(T) == 4 ? 8 : 4;
  uint4 a[kPieces], b[kPieces];
  uint16_t e;
  __device__ __forceinline__ void load(const uint8_t* block, int lane) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      a[j] = *reinterpret_cast<const uint4*>(block + j * 512 + lane * 16);
      b[j] = *reinterpret_cast<const uint4*>(block + kPieces * 512 + j * 512 + lane * 16);
    }
    e = sizeof(T) == 4 ? 0 : reinterpret_cast<const uint16_t*>(block + 4096)[lane];
  }
  __device__ __forceinline__ void decode(float (&g)[32], float (&u)[32]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[4 * j] = __uint_as_float(a[j].x); g[4 * j + 1] = __uint_as_float(a[j].y);
        g[4 * j + 2] = __uint_as_float(a[j].z); g[4 * j + 3] = __uint_as_float(a[j].w);
        u[4 * j] = __uint_as_float(b[j].x); u[4 * j + 1] = __uint_as_float(b[j].y);
        u[4 * j + 2] = __uint_as_float(b[j].z); u[4 * j + 3] = __uint_as_float(b[j].w);
      }
    } else {
      // the exponents as signed bytes; -100 and up, so 2^(e - 14) is a normal number
      const float sg = exp2_int((int)(int8_t)(e & 0xff) - 14), su = exp2_int((int)(int8_t)(e >> 8) - 14);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t aw[4] = {a[j].x, a[j].y, a[j].z, a[j].w}, bw[4] = {b[j].x, b[j].y, b[j].z, b[j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&aw[k]));
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&bw[k]));
          g[8 * j + 2 * k] = x.x * sg; g[8 * j + 2 * k + 1] = x.y * sg;
          u[8 * j + 2 * k] = y.x * su; u[8 * j + 2 * k + 1] = y.y * su;
        }
      }
    }
  }
};

// Lane l returns the sum over the warp's lanes of v[l]: 31 shuffles, in an
// order fixed by the lanes.
__device__ __forceinline__ float column_sum32(float (&v)[32], int lane) {
#pragma unroll
  for (int half = 16; half; half >>= 1) {
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
// How the last R tiles of a product are cut along their nkb K blocks among W
// workers.  Worker s R + t, s < S: slice s of tile t, K blocks [s a, s a + a).
// The E = W - S R others: equal runs of the units (tile, K block >= S a), tile
// after tile.  Slots: the worker's index in the first case; S R + e + t in the
// second (unique, since along the runs either e or t grows by one).
struct Cut {
  int R, S, E, a, nkb;
  __host__ __device__ Cut(int R_, int W, int nkb_) : R(R_), nkb(nkb_) {
    S = W / R;
    E = W - S * R;
    a = E ? (int)((int64_t)nkb * R / W) : (nkb + S - 1) / S;
  }
  __host__ __device__ int rest() const { return E ? nkb - S * a : 0; }  // K blocks of the runs
  __host__ __device__ int slots() const { return S * R + (E ? E + R : 0); }
};

struct Work {
  int worker, workers, nkb;
  int at, whole_end;            // whole tiles: at, at + workers, ... below whole_end
  int base;                     // first of the cut tiles; -1: none
  int64_t unit, unit_end;       // units still to do of a run
  bool slice;                   // the slice is still to do
  int tile, kb0, kb1, slot;     // the current piece; slot < 0: a whole tile
  __device__ __forceinline__ Work(const GemmArgs& a, int worker_, int workers_)
      : worker(worker_), workers(workers_), nkb(a.nk * a.nseg), at(worker_), base(-1), unit(0), unit_end(0), slice(false) {
    const int tiles = a.tiles_m * a.tiles_n * a.batches;
    whole_end = tiles;
    if (a.split) {
      base = whole_end = tiles / workers * workers;
      const Cut c(tiles - base, workers, nkb);
      slice = worker < c.S * c.R;
      if (!slice) {
        const int e = worker - c.S * c.R;
        const int64_t units = (int64_t)c.R * c.rest();
        unit = units * e / c.E;
        unit_end = units * (e + 1) / c.E;
      }
    }
  }
  __device__ __forceinline__ bool next(const GemmArgs& a) {
    if (at < whole_end) {
      tile = at;
      at += workers;
      kb0 = 0;
      kb1 = nkb;
      slot = -1;
      return true;
    }
    if (base < 0) return false;
    const Cut c(a.tiles_m * a.tiles_n * a.batches - base, workers, nkb);
    if (slice) {
      slice = false;
      const int s = worker / c.R;
      tile = base + worker - s * c.R;
      kb0 = s * c.a;
      kb1 = min(nkb, kb0 + c.a);
      slot = worker;
      return kb0 < kb1;
    }
    if (unit >= unit_end) return false;
    const int rest = c.rest();
    const int t = (int)(unit / rest);
    const int k = (int)(unit - (int64_t)t * rest);
    const int len = (int)min((int64_t)(rest - k), unit_end - unit);
    tile = base + t;
    kb0 = c.S * c.a + k;
    kb1 = kb0 + len;
    slot = c.S * c.R + (worker - c.S * c.R) + t;
    unit += len;
    return true;
  }
};

// Tile index -> (batch, row tile, column tile): blocks of group_m row tiles,
// row tiles fastest inside a block, so the CTAs of a wave share both operands
// in the L2.
__device__ __forceinline__ void tile_at(const GemmArgs& a, int tile, int& z, int& mt, int& nt) {
  const int per = a.tiles_m * a.tiles_n;
  z = tile / per;
  int t = tile - z * per;
  const int block = t / (a.group_m * a.tiles_n);
  const int rows = min(a.group_m, a.tiles_m - block * a.group_m);
  t -= block * a.group_m * a.tiles_n;
  nt = t / rows;
  mt = block * a.group_m + (t - nt * rows);
}

// ---------------------------------------------------------------- kernel
template <typename T, int EPI, int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(NTHREADS, 1)
ffn_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ GemmArgs a) {
  constexpr int S = stages(BN);
  constexpr uint32_t STAGE = stage_bytes(BN);
  constexpr bool GATED = EPI == EPI_GATED;
  constexpr int COLS = GATED ? BN / 2 : BN;  // output columns of a tile
  constexpr bool WIDE = sizeof(T) == 4;
  // K blocks of one accumulation in TMEM.  The tensor cores truncate each
  // addition to the accumulator, an error that grows with the number of steps
  // (measured on fp32 data: 2.4e-6 of the result's norm after 128 steps, where
  // sums rounded to nearest leave 6e-7); fp32 data therefore moves its sums to
  // registers every kWideRun blocks.  16-bit results do not see the difference.
  constexpr int RUN = WIDE ? kWideRun : 1 << 30;
  static_assert(!WIDE || BN <= 128, "an epilogue thread holds BN / 2 sums");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_addr(smem);
  uint8_t* staging = smem + S * STAGE;
  uint8_t* tail = staging + kStaging + EPI_WARPS * 64 * 4;
  if (smem + smem_bytes(BN) > smem_raw + smem_bytes(BN) + kSmemSlack) {  // an unexpected start: nothing is touched
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
  constexpr uint32_t TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(smem_addr(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Work w(a, blockIdx.x, gridDim.x);

  if (warp == LOAD_WARP) {
    // ------------------------------------------------ TMA loads
    if (lane == 0) {
      int issued = 0;
      bool ok = true;
      while (ok && w.next(a)) {
        int z, mt, nt;
        tile_at(a, w.tile, z, mt, nt);
        const int m0 = mt * BM, n0 = nt * COLS;
        int sg = w.kb0 / a.nk, kb = w.kb0 - sg * a.nk;
        for (int i = w.kb0; i < w.kb1; ++i) {
          const int s = issued % S;
          ok = mbar_wait(empty(s), ((issued / S) & 1) ^ 1, abort_flag, a.status, ST_FFN_LOAD);
          if (!ok) break;
          const Seg seg = a.seg[sg];
          const int k = kb * BK;
          const uint32_t dst = sbase + s * STAGE;
          const CUtensorMap* ma = &maps.m[seg.a_map + z];
          const CUtensorMap* mb = &maps.m[seg.b_map];
          mbar_arrive_expect_tx(full(s), STAGE);
          if (A_MN) {
            tma_load_3d(dst, ma, m0, k, seg.a_plane, full(s));
            tma_load_3d(dst + 8192, ma, m0 + 64, k, seg.a_plane, full(s));
          } else {
            tma_load_3d(dst, ma, k, m0, seg.a_plane, full(s));
          }
          if (GATED) {
            tma_load_3d(dst + A_STAGE, mb, k, n0, seg.b_plane, full(s));
            tma_load_3d(dst + A_STAGE + COLS * 128, mb + 1, k, n0, seg.b_plane, full(s));
          } else if (B_MN) {
#pragma unroll
            for (int q = 0; q < BN / 64; ++q)
              tma_load_3d(dst + A_STAGE + q * 8192, mb, n0 + 64 * q, k, seg.b_plane, full(s));
          } else {
            tma_load_3d(dst + A_STAGE, mb, k, n0, seg.b_plane, full(s));
          }
          ++issued;
          if (++kb == a.nk) {
            kb = 0;
            ++sg;
          }
        }
      }
      // copies in flight land before the CTA may go
      for (int i = issued > S ? issued - S : 0; i < issued; ++i)
        mbar_wait(full(i % S), (i / S) & 1, abort_flag, a.status, ST_FFN_DRAIN);
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t idesc = tcc::idesc_f16_major(BM, BN, a.operand_bf16 != 0, A_MN, B_MN);
      int used = 0, done = 0;
      bool ok = true;
      while (ok && w.next(a)) {
        for (int k0 = w.kb0; ok && k0 < w.kb1; k0 += RUN) {
          const int k1 = w.kb1 - k0 > RUN ? k0 + RUN : w.kb1;
          const int b = done & 1;
          ok = mbar_wait(acc_empty(b), ((done >> 1) & 1) ^ 1, abort_flag, a.status, ST_FFN_MMA);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(b * BN);
          for (int i = k0; i < k1; ++i) {
            const int s = used % S;
            ok = mbar_wait(full(s), (used / S) & 1, abort_flag, a.status, ST_FFN_MMA);
            if (!ok) break;
            tc_fence_after();
            const uint32_t ab = sbase + s * STAGE, bb = ab + A_STAGE;
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              const uint64_t ad = A_MN ? tcc::desc_mnmajor_sw128(ab + kk * 2048, 8192) : desc_kmajor_sw128(ab + kk * 32);
              const uint64_t bd = B_MN ? tcc::desc_mnmajor_sw128(bb + kk * 2048, 8192) : desc_kmajor_sw128(bb + kk * 32);
              mma_f16(d, ad, bd, idesc, (i > k0 || kk > 0) ? 1u : 0u);
            }
            mma_commit(empty(s));
            ++used;
          }
          if (!ok) break;
          mma_commit(acc_full(b));
          ++done;
        }
      }
      // MMAs still running finish before TMEM and shared memory are released
      if (used > 0) {
        mma_commit(drain);
        mbar_wait(drain, 0, abort_flag, a.status, ST_FFN_DRAIN);
      }
    }
  } else {
    // ------------------------------------------------ epilogue
    const int q = warp & 3, half = warp >> 2;
    // the bias values of a 32-column block, one column a lane, read back by all
    // lanes; each warp has its own, so the epilogue warps never meet at a barrier
    float* colf = reinterpret_cast<float*>(staging + kStaging) + warp * 64;
    auto bias32 = [&](int c0) {
      __syncwarp();
#pragma unroll
      for (int k = 0; k < (GATED ? 2 : 1); ++k)
        colf[k * 32 + lane] = c0 + lane < a.N ? to_f<T>(static_cast<const T*>(a.bias[k])[c0 + lane]) : 0.0f;
      __syncwarp();
    };
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    uint8_t* stage = staging + warp * (2 * kStageBlock);
    const bool has_bias = EPI != EPI_DGATE && a.bias[0] != nullptr;
    const int64_t col_blocks = (a.N + 31) / 32;
    // this warp's staged blocks, out through the TMA
    auto store_staged = [&](int blocks, int x, int y, int first) {
      fence_async_shared();
      __syncwarp();
      if (lane == 0 && y < a.M) {
        for (int k = 0; k < blocks; ++k)
          tma_store_3d(&maps.out[first + k], smem_addr(stage + k * kStageBlock), x, y, 0);
        bulk_commit();
      }
    };
    // staged blocks may be written again once the store has read them
    auto staging_free = [&] {
      if (lane == 0) bulk_wait_read_all();
      __syncwarp();
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
      if (lane == 0) mbar_arrive(acc_empty(done & 1));
      ++done;
    };
    while (ok && w.next(a)) {
      int z, mt, nt;
      tile_at(a, w.tile, z, mt, nt);
      const int n0 = nt * COLS;
      const int row0 = mt * BM + q * 32;
      const int64_t row = (int64_t)row0 + lane;
      const bool row_in = row < a.M;
      const bool whole = w.slot < 0;
      const int64_t m_block = (int64_t)mt * 4 + q;
      auto saved_block = [&](int c) {
        return static_cast<uint8_t*>(a.saved) + saved_block_offset<T>(m_block, (n0 + c * 32) / 32, col_blocks);
      };

      // one 32-column block of this tile; v, u: the sums of its columns (GATED: gate and up)
      auto block = [&](int c, float (&v)[32], float (&u)[32], const SavedRaw<T>& raw) {
        const int c0 = n0 + c * 32;
        if (!whole) {
          // an fp32 partial of this tile, 16-byte pieces of 32 rows side by side
          float* slot = a.partial + (int64_t)w.slot * (BM * BN) + q * (32 * BN);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(slot + c * 1024 + j * 128 + lane * 4) =
                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          return;
        }
        if (c0 >= a.N) return;
        if (has_bias) {
          bias32(c0);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            v[j] += colf[j];
            if (GATED) u[j] += colf[32 + j];
          }
        }
        if constexpr (EPI == EPI_GATED) {
          if (a.saved) save_gate_up<T>(saved_block(c), lane, v, u);
          float h[32];
          gate32<WIDE>(a.act, v, u, h);
          if constexpr (WIDE) {
            if (row_in) store_operand32<T>(a.out[0], a.plane, row, a.ldo, c0, h);
          } else {
            staging_free();
            stage_row32<T>(stage, lane, h);
            store_staged(1, c0, row0, 0);
          }
        } else if constexpr (EPI == EPI_DGATE) {
          // rows past M: their saved values are those of zero rows, and dh is 0
          float g[32], d[32];
          raw.decode(g, d);
          dgate32<WIDE>(a.act, v, g, d);
          if constexpr (WIDE) {
            if (row_in) {
              store_operand32<T>(a.out[0], a.plane, row, a.ldo, c0, g);
              store_operand32<T>(a.out[1], a.plane, row, a.ldo, c0, d);
            }
          } else {
            staging_free();
            stage_row32<T>(stage, lane, g);
            stage_row32<T>(stage + kStageBlock, lane, d);
            store_staged(2, c0, row0, 0);
          }
          if (a.colsum) {
            if (!row_in) {
#pragma unroll
              for (int j = 0; j < 32; ++j) g[j] = d[j] = 0.0f;
            }
            const float sg = column_sum32(g, lane), su = column_sum32(d, lane);
            if (c0 + lane < a.N) {
              float* out = a.colsum + (m_block * 2) * a.N + c0 + lane;
              out[0] = sg;
              out[a.N] = su;
            }
          }
        } else {
          if (!WIDE && a.vec) {
            if constexpr (!WIDE) {
              staging_free();
              stage_row32<T>(stage, lane, v);
              store_staged(1, c0, row0, z);
            }
          } else if (row_in) {
            store_row32<T>(static_cast<T*>(a.out[z]) + row * a.ldo, c0, a.N, a.vec != 0, v);
          }
        }
      };

      SavedRaw<T> raw;
      if constexpr (WIDE) {
        // this thread's columns: blocks half, half + 2, ...; at most two of them (BN = 128)
        constexpr int NB = (GATED ? COLS / 32 : BN / 32) > 2 ? 2 : 1;
        float sum[NB][32], sum_u[GATED ? NB : 1][32];
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            sum[k][j] = 0.0f;
            if (GATED) sum_u[k][j] = 0.0f;
          }
        for (int k0 = w.kb0; k0 < w.kb1; k0 += RUN) {
          if (!wait_acc()) break;
          const uint32_t acc = lanes + (uint32_t)((done & 1) * BN);
#pragma unroll
          for (int k = 0; k < NB; ++k) {
            const int c = half + 2 * k;
            if (c * 32 >= COLS) break;
            float t[32];
            tmem_ld32(acc + c * 32, t);
            tmem_ld32_wait(t);
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[k][j] += t[j];
            if constexpr (GATED) {
              tmem_ld32(acc + COLS + c * 32, t);
              tmem_ld32_wait(t);
#pragma unroll
              for (int j = 0; j < 32; ++j) sum_u[k][j] += t[j];
            }
          }
          release_acc();
        }
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const int c = half + 2 * k;
          if (c * 32 >= COLS) break;
          if (EPI == EPI_DGATE && n0 + c * 32 < a.N) raw.load(saved_block(c), lane);
          block(c, sum[k], sum_u[GATED ? k : 0], raw);
        }
      } else {
        // the first block's saved values are fetched while the products run, the next ones' a block ahead
        if (EPI == EPI_DGATE && n0 + half * 32 < a.N) raw.load(saved_block(half), lane);
        if (!wait_acc()) break;
        const uint32_t acc = lanes + (uint32_t)((done & 1) * BN);
#pragma unroll 1
        for (int c = half; c < COLS / 32; c += 2) {
          float v[32], u[32];
          tmem_ld32(acc + c * 32, v);
          if (GATED) tmem_ld32(acc + COLS + c * 32, u);
          tmem_ld32_wait(v);
          if (GATED) tmem_ld32_wait(u);
          const SavedRaw<T> now = raw;
          if (EPI == EPI_DGATE && c + 2 < COLS / 32 && n0 + (c + 2) * 32 < a.N) raw.load(saved_block(c + 2), lane);
          block(c, v, u, now);
        }
        release_acc();
      }
    }
    // the stores have left shared memory and are done before the CTA ends
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace ffn
}  // namespace dcn
