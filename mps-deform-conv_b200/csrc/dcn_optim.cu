// dcn_optim.cu -- the optimizer step of a network's parameters: one AdamW step
// over many tensors, and the global gradient norm whose clipping factor that
// step reads from device memory.
//
// AdamW with decoupled weight decay, t = steps taken + 1, g = grad * grad_scale:
//   m' = b1 m + (1 - b1) g          v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
// All arithmetic is fp32 (the bias corrections fp64); m and v are updated with
// one rounding per product and sum, so a state does not depend on how the
// compiler contracts them.  A 16-bit parameter is rounded once, from the fp32
// result; with a master copy the fp32 result is kept and the parameter is its
// rounding.
//
// 8-bit states.  m, and sqrt(v) (which halves the decades v spans), are held
// as float8 e4m3 codes with one fp32 scale per 256 elements of the tensor:
//   e = clamp(floor(log2 max|x|), -100, 127), scale = 2^(e - 7), code = x / scale
// so the largest element lands in [128, 256) and the products with the scale
// are exact.  The code is rounded stochastically: a 16-bit word, a hash of the
// element's index, the step and the seed, is added below the last kept bit.
// Rounding to nearest would freeze v: with b2 = 0.999 one step moves sqrt(v)
// by at most 0.05 % while e4m3's steps are 6 to 12 %.  A positive sqrt(v) never
// becomes code 0, which would leave m' over eps alone.
//
// What bounds it: HBM.  Every element is read and written once (28 bytes for a
// bf16 parameter with a master copy and fp32 states, 10 with 8-bit states and
// none), and nothing is reused.  A warp takes 256 consecutive elements, eight
// per lane, as 16-byte loads where every pointer of the tensor allows them and
// as single elements, 32 lanes side by side, where not and at tails.
// Measured on 96.6 M bf16 parameters: fp32 states with master copies 415 us, the
// measured copy rate; 8-bit states without 293 us, 3.3 TB/s: some 80
// instructions an element (exact root, two codes, hash) hold it there.
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include <cuda_fp8.h>

#include "dcn_optim.h"

namespace dcn {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBlockElems = 256;                          // elements of one 8-bit scale, and of one warp pass
constexpr int kRow = kWarps * kBlockElems;                // elements of one pass of a CTA
// Passes of a CTA, at most: its prologue (the counters, the powers) is paid once
// and 8-bit passes are fetched ahead; 32-bit states run at the memory's rate and
// only pay for the longer tail (421 us at 4, 443 at 16 for 96.6 M bf16 parameters
// with master copies; 8 bits: 454 at 4, 288 at 16).
constexpr int kMostPasses = 16;

struct AdamwEntry {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* exp_avg_scale;
  float* exp_avg_sq_scale;
  float* master;
  int32_t* step;
  long long numel;
  uint32_t first_chunk;
  uint16_t vec;       // every pointer allows 16-byte access
  uint16_t advance;   // the last use of this step counter in the call
};

struct AdamwHyper {
  double lr, beta1, beta2, weight_decay;
  float b1, omb1, b2, omb2, eps;
  const float* lr_device;
  const float* grad_scale;
  uint32_t seed;
};

// Entries travel in the kernel's arguments (at most 32,764 bytes): no device
// table to fill, so a call is one launch and can be captured into a graph.
template <int N>
struct AdamwArgs {
  AdamwHyper h;
  uint32_t n;
  int passes;  // of a CTA: a chunk is passes x kRow elements
  AdamwEntry e[N];
};

// The published 32-bit integer hash with the "lowbias32" constants (C. Wellons).
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

// Codes of a block's values, |x| < 2^(e + 1): x / 2^(e - 7) scaled by 2^-120 on
// top, which puts e4m3's smallest normal 2^-6 at fp32's 2^-126, so that the top
// bits of the fp32 pattern (subnormals included) are the code, and adding a word
// below bit 20 before they are cut off rounds up with the remainder's
// probability.  The two factors are one where 2^(-113 - e) is a normal number.
struct CodeScale {
  float first, second;
  bool two, check;  // of the whole warp; check: the block holds inf or NaN
  __device__ __forceinline__ CodeScale(int e, bool check_) : check(check_) {
    two = e > 13;
    first = __int_as_float((two ? 7 - e + 127 : -113 - e + 127) << 23);
    second = two ? 7.5231638452626401e-37f : 1.0f;  // 2^-120
  }
  __device__ __forceinline__ uint32_t operator()(float x, uint32_t word16) const {
    float z = __fmul_rn(fabsf(x), first);
    if (two) z = __fmul_rn(z, second);
    uint32_t code = (__float_as_uint(z) + (word16 << 4)) >> 20;
    if (check && !(fabsf(x) <= 3.402823466e38f)) code = 0x7f;
    return code;
  }
};

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;
}
// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// The block's exponent from the lanes' largest values (NaN kept: patterns of
// non-negative floats, inf and NaN order as integers do); `bad`: not all finite.
__device__ __forceinline__ int block_exponent(float top, const float (&x)[8], bool& bad) {
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);
  bad = bits >= 0x7f800000u;
  if (bad) {  // the finite values' exponent
    float t = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) t = fmaxf(t, finite_abs(x[j]));
    bits = __reduce_max_sync(0xffffffffu, __float_as_uint(t));
  }
  return max(-100, (int)(bits >> 23) - 127);
}

// Two fp32 products an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 twice(float a) { return make_float2(a, a); }
// m / d for a positive normal d: the reciprocal is off by at most one unit in
// the last place.
__device__ __forceinline__ float rcp_fast(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

__device__ __forceinline__ float2 e4m3_pair(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}

// Eight elements of a tensor of element type T, and as floats.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    T t[8];
    memcpy(t, v, sizeof(t));
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = to_f<T>(t[j]);
  }
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  Raw8<T> r;
  r.load(p);
  r.get(v);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_f<T>(v[j]);
    uint4 a;
    memcpy(&a, t, 16);
    *reinterpret_cast<uint4*>(p) = a;
  }
}

// What a lane reads of a whole, aligned pass; fetched a pass ahead.
template <typename T, bool MASTER, bool BITS8>
struct AdamwRaw {
  Raw8<T> g;
  Raw8<std::conditional_t<MASTER, float, T>> p;
  Raw8<float> m, v;   // 32-bit states
  uint2 mc, vc;       // 8-bit states
  float sm, sv;
  __device__ __forceinline__ void load(const AdamwEntry& t, long long base, int lane) {
    const long long i = base + 8 * lane;
    g.load(static_cast<const T*>(t.grad) + i);
    if constexpr (MASTER) p.load(t.master + i);
    else p.load(static_cast<const T*>(t.param) + i);
    if constexpr (BITS8) {
      mc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.exp_avg) + i);
      vc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.exp_avg_sq) + i);
      sm = t.exp_avg_scale[base / kBlockElems];
      sv = t.exp_avg_sq_scale[base / kBlockElems];
    } else {
      m.load(static_cast<const float*>(t.exp_avg) + i);
      v.load(static_cast<const float*>(t.exp_avg_sq) + i);
    }
  }
};

// One warp's pass over elements [base, base + 256) of tensor `t`.
template <typename T, bool MASTER, bool BITS8, bool VEC>
__device__ __forceinline__ void adamw_pass(const AdamwEntry& t, const AdamwHyper& h, long long base, int lane,
                                           float gs, float decay, float step_size, float corr, uint32_t key,
                                           const AdamwRaw<T, MASTER, BITS8>& raw) {
  // lane's element j: VEC base + 8 lane + j, else base + lane + 32 j
  auto at = [&](int j) { return VEC ? base + 8 * lane + j : base + lane + 32 * j; };
  float g[8], p[8], m[8], r[8];   // r: v, then sqrt(v')
  const T* grad = static_cast<const T*>(t.grad);
  T* param = static_cast<T*>(t.param);
  float* mf = static_cast<float*>(t.exp_avg);
  float* vf = static_cast<float*>(t.exp_avg_sq);
  uint8_t* mc = static_cast<uint8_t*>(t.exp_avg);
  uint8_t* vc = static_cast<uint8_t*>(t.exp_avg_sq);
  const long long blk = base / kBlockElems;
  if (VEC) {
    raw.g.get(g);
    raw.p.get(p);
    if constexpr (BITS8) {
      const uint32_t aw[4] = {raw.mc.x, raw.mc.x >> 16, raw.mc.y, raw.mc.y >> 16};
      const uint32_t bw[4] = {raw.vc.x, raw.vc.x >> 16, raw.vc.y, raw.vc.y >> 16};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = mul2(e4m3_pair(aw[j]), twice(raw.sm)), y = mul2(e4m3_pair(bw[j]), twice(raw.sv));
        const float2 q = mul2(y, y);
        m[2 * j] = x.x; m[2 * j + 1] = x.y;
        r[2 * j] = q.x; r[2 * j + 1] = q.y;
      }
    } else {
      raw.m.get(m);
      raw.v.get(r);
    }
  } else {
    const float sm = BITS8 ? t.exp_avg_scale[blk] : 1.0f, sv = BITS8 ? t.exp_avg_sq_scale[blk] : 1.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long i = at(j);
      const bool in = i < t.numel;
      g[j] = in ? to_f<T>(grad[i]) : 0.0f;
      p[j] = in ? (MASTER ? t.master[i] : to_f<T>(param[i])) : 0.0f;
      if (BITS8) {
        m[j] = in ? __fmul_rn(e4m3_pair(mc[i]).x, sm) : 0.0f;
        const float y = in ? __fmul_rn(e4m3_pair(vc[i]).x, sv) : 0.0f;
        r[j] = __fmul_rn(y, y);
      } else {
        m[j] = in ? mf[i] : 0.0f;
        r[j] = in ? vf[i] : 0.0f;
      }
    }
  }

  float mtop = 0.0f, rtop = 0.0f;
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    // scalar intrinsics: products and sums in pairs (f32x2) may be fused
    const float gk = __fmul_rn(g[k], gs);
    m[k] = __fadd_rn(__fmul_rn(m[k], h.b1), __fmul_rn(gk, h.omb1));
    v[k] = __fadd_rn(__fmul_rn(r[k], h.b2), __fmul_rn(__fmul_rn(gk, gk), h.omb2));
    r[k] = __fsqrt_rn(v[k]);
    p[k] = p[k] * decay - step_size * (m[k] * rcp_fast(r[k] * corr + h.eps));
    if (BITS8) {
      mtop = max_nan(mtop, fabsf(m[k]));
      rtop = max_nan(rtop, r[k]);
    }
  }

  uint32_t cm[8], cr[8];
  if (BITS8) {
    bool bad_m, bad_r;
    const int em = block_exponent(mtop, m, bad_m), er = block_exponent(rtop, r, bad_r);
    if (lane == 0) {
      t.exp_avg_scale[blk] = pow2i(em - 7);
      t.exp_avg_sq_scale[blk] = pow2i(er - 7);
    }
    const CodeScale qm(em, bad_m), qr(er, bad_r);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = mix32((uint32_t)at(j) ^ key);
      cm[j] = qm(m[j], w & 0xffffu) | ((__float_as_uint(m[j]) >> 24) & 0x80u);
      // a positive root keeps at least the smallest code
      cr[j] = max(qr(r[j], w >> 16), min(__float_as_uint(r[j]), 1u));
    }
  }

  if (VEC) {
    const long long i = base + 8 * lane;
    store8<T>(param + i, p);
    if (MASTER) store8<float>(t.master + i, p);
    if (BITS8) {
      *reinterpret_cast<uint2*>(mc + i) = make_uint2(cm[0] | cm[1] << 8 | cm[2] << 16 | cm[3] << 24,
                                                     cm[4] | cm[5] << 8 | cm[6] << 16 | cm[7] << 24);
      *reinterpret_cast<uint2*>(vc + i) = make_uint2(cr[0] | cr[1] << 8 | cr[2] << 16 | cr[3] << 24,
                                                     cr[4] | cr[5] << 8 | cr[6] << 16 | cr[7] << 24);
    } else {
      store8<float>(mf + i, m);
      store8<float>(vf + i, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long i = at(j);
      if (i >= t.numel) continue;
      param[i] = from_f<T>(p[j]);
      if (MASTER) t.master[i] = p[j];
      if (BITS8) {
        mc[i] = (uint8_t)cm[j];
        vc[i] = (uint8_t)cr[j];
      } else {
        mf[i] = m[j];
        vf[i] = v[j];
      }
    }
  }
}

// b^n in fp64 by squaring: at most 62 products where pow takes some 2 us; the
// relative error, below n 2^-52, is far below what an fp32 correction keeps.
__device__ __forceinline__ double power(double b, uint32_t n) {
  double r = 1.0;
#pragma unroll 1
  for (; n; n >>= 1) {
    if (n & 1) r *= b;
    b *= b;
  }
  return r;
}

template <typename T, bool MASTER, bool BITS8, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ AdamwArgs<N> a) {
  __shared__ float s_bias[3];     // decay, step size, 1 / sqrt(1 - b2^t)
  __shared__ uint32_t s_key;
  __shared__ bool s_last;
  const AdamwHyper& h = a.h;
  // the tensor of this CTA's chunk: the last entry that starts at or before it
  uint32_t lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) >> 1;
    if (a.e[mid].first_chunk <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const AdamwEntry& t = a.e[lo];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long start = (long long)(blockIdx.x - t.first_chunk) * a.passes * kRow + warp * kBlockElems;
  auto whole = [&](int i) { return i < a.passes && t.vec && start + (long long)i * kRow + kBlockElems <= t.numel; };
  AdamwRaw<T, MASTER, BITS8> raw;
  // 32-bit states have enough in flight without it, and lose more by the registers
  if (BITS8 && whole(0)) raw.load(t, start, lane);
  if (lane == 0 && warp < 2) {  // the two corrections side by side
    const int step = t.step[0] + 1;
    const double lr = h.lr_device ? (double)*h.lr_device : h.lr;
    const double left = 1.0 - power(warp == 0 ? h.beta1 : h.beta2, (uint32_t)step);
    if (warp == 0) {
      s_bias[0] = (float)(1.0 - lr * h.weight_decay);
      s_bias[1] = (float)(lr / left);
      s_key = mix32(h.seed + (uint32_t)step * 0x9e3779b9u);
    } else {
      s_bias[2] = (float)rsqrt(left);
    }
  }
  // not finite: the whole step is skipped, nothing is written
  const float gs = h.grad_scale ? *h.grad_scale : 1.0f;
  __syncthreads();
  if (!(fabsf(gs) <= 3.402823466e38f)) return;
  const float decay = s_bias[0], step_size = s_bias[1], corr = s_bias[2];
  const uint32_t key = s_key;
#pragma unroll 1
  for (int i = 0; i < a.passes; ++i) {
    const long long base = start + (long long)i * kRow;
    if (base >= t.numel) break;
    if (whole(i)) {
      if (!BITS8) raw.load(t, base, lane);
      const AdamwRaw<T, MASTER, BITS8> now = raw;
      if (BITS8 && whole(i + 1)) raw.load(t, base + kRow, lane);
      adamw_pass<T, MASTER, BITS8, true>(t, h, base, lane, gs, decay, step_size, corr, key, now);
    } else {
      adamw_pass<T, MASTER, BITS8, false>(t, h, base, lane, gs, decay, step_size, corr, key, raw);
    }
  }

  // every CTA has read its step counter before it takes a ticket, so the last
  // one may advance the counters; the ticket (the first tensor's step[1]) goes
  // back to zero for the next call
  __syncthreads();
  if (threadIdx.x == 0) {
    const int ticket = atomicAdd(&a.e[0].step[1], 1);
    s_last = ticket == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  for (uint32_t i = threadIdx.x; i < a.n; i += kThreads)
    if (a.e[i].advance) a.e[i].step[0] += 1;
  if (threadIdx.x == 0) a.e[0].step[1] = 0;
}

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

template <typename T, bool MASTER, bool BITS8, int N>
cudaError_t adamw_launch(const AdamwHyper& h, const AdamwEntry* e, uint32_t n, uint32_t chunks, int passes,
                         cudaStream_t st) {
  AdamwArgs<N> a;
  a.h = h;
  a.n = n;
  a.passes = passes;
  std::copy(e, e + n, a.e);
  KernelScope ks("adamw", st);
  adamw_kernel<T, MASTER, BITS8, N><<<std::max(1u, chunks), kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

// Entries of a launch: a layer's tensors, some, many, or what 32,764 bytes of
// arguments hold; the arguments of a small call take less time to send.
constexpr int kLarge = 384;
static_assert(sizeof(AdamwArgs<kLarge>) <= 32764, "kernel arguments");

template <typename T, bool MASTER, bool BITS8>
cudaError_t adamw_group(const AdamwHyper& h, const std::vector<AdamwEntry>& all, cudaStream_t st) {
  // as many passes a CTA as leave eight CTAs an SM
  unsigned long long total = 0;
  for (const AdamwEntry& e : all) total += (unsigned long long)e.numel;
  const int passes = (int)std::min<unsigned long long>(BITS8 ? kMostPasses : kMostPasses / 4, std::max<unsigned long long>(1, total / (kRow * 148ull * 8)));
  const unsigned long long chunk = (unsigned long long)passes * kRow;
  // launches of at most kLarge tensors and 2^31 - 1 chunks (first_chunk restarts in each)
  size_t i = 0;
  while (i < all.size()) {
    std::vector<AdamwEntry> part;
    unsigned long long chunks = 0;
    while (i < all.size() && part.size() < (size_t)kLarge) {
      const unsigned long long c = ((unsigned long long)all[i].numel + chunk - 1) / chunk;
      if (!part.empty() && chunks + c > 0x7fffffffull) break;
      part.push_back(all[i]);
      part.back().first_chunk = (uint32_t)chunks;
      chunks += c;
      ++i;
    }
    auto go = [&](auto cap) {
      return adamw_launch<T, MASTER, BITS8, decltype(cap)::value>(h, part.data(), (uint32_t)part.size(), (uint32_t)chunks,
                                                                  passes, st);
    };
    const cudaError_t e = part.size() <= 12   ? go(std::integral_constant<int, 12>{})
                          : part.size() <= 48 ? go(std::integral_constant<int, 48>{})
                          : part.size() <= 144 ? go(std::integral_constant<int, 144>{})
                                               : go(std::integral_constant<int, kLarge>{});
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t adamw_step(const dcn_adamw_options& o, const dcn_adamw_tensor* t, int64_t n, cudaStream_t st) {
  AdamwHyper h;
  h.lr = o.lr; h.beta1 = o.beta1; h.beta2 = o.beta2; h.weight_decay = o.weight_decay;
  h.b1 = (float)o.beta1; h.omb1 = (float)(1.0 - o.beta1);
  h.b2 = (float)o.beta2; h.omb2 = (float)(1.0 - o.beta2);
  h.eps = (float)o.eps;
  h.lr_device = o.lr_device;
  h.grad_scale = o.grad_scale;
  h.seed = o.seed;
  // one launch group per (dtype, master copies or not): entries in call order
  std::vector<AdamwEntry> group[3][2];
  for (int64_t i = 0; i < n; ++i) {
    AdamwEntry e;
    e.param = t[i].param; e.grad = t[i].grad; e.exp_avg = t[i].exp_avg; e.exp_avg_sq = t[i].exp_avg_sq;
    e.exp_avg_scale = t[i].exp_avg_scale; e.exp_avg_sq_scale = t[i].exp_avg_sq_scale;
    e.master = t[i].master; e.step = t[i].step; e.numel = t[i].numel;
    e.first_chunk = 0;
    const size_t state = o.state_bits == 8 ? 8 : 16;
    e.vec = aligned(e.param, 16) && aligned(e.grad, 16) && aligned(e.exp_avg, state) && aligned(e.exp_avg_sq, state) &&
            aligned(e.master, 16);
    e.advance = 0;
    group[t[i].dtype][e.master != nullptr].push_back(e);
  }
  // a counter is advanced by its last use, in launch order
  std::vector<int32_t*> seen;
  for (int d = 2; d >= 0; --d)
    for (int m = 1; m >= 0; --m)
      for (size_t i = group[d][m].size(); i-- > 0;) seen.push_back(group[d][m][i].step);
  {
    std::vector<std::pair<int32_t*, size_t>> order(seen.size());
    for (size_t i = 0; i < seen.size(); ++i) order[i] = {seen[i], i};
    std::sort(order.begin(), order.end());
    std::vector<char> first(seen.size(), 0);
    for (size_t i = 0; i < order.size(); ++i)
      if (i == 0 || order[i].first != order[i - 1].first) first[order[i].second] = 1;
    size_t k = 0;
    for (int d = 2; d >= 0; --d)
      for (int m = 1; m >= 0; --m)
        for (size_t i = group[d][m].size(); i-- > 0;) group[d][m][i].advance = first[k++];
  }
  cudaError_t err = cudaSuccess;
  auto run = [&](int dtype, bool master) {
    const auto& g = group[dtype][master];
    if (g.empty() || err != cudaSuccess) return;
    auto pick = [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      if (o.state_bits == 8) err = master ? adamw_group<T, true, true>(h, g, st) : adamw_group<T, false, true>(h, g, st);
      else err = master ? adamw_group<T, true, false>(h, g, st) : adamw_group<T, false, false>(h, g, st);
    };
    if (dtype == DCN_FLOAT32) pick((float*)nullptr);
    else if (dtype == DCN_FLOAT16) pick((__half*)nullptr);
    else pick((__nv_bfloat16*)nullptr);
  };
  for (int d = 0; d < 3; ++d)
    for (int m = 0; m < 2; ++m) run(d, m != 0);
  return err;
}

// ---------------------------------------------------------------- gradient norm
// norm = sqrt(sum of all squares) / loss_scale.  Each CTA sums its share of the
// chunks in a fixed order and writes one fp64 partial; a second one-CTA kernel
// adds the partials in order, so the result does not depend on timing.  HBM
// bound: the gradients are read once (96.6 M bf16 values: 39 us, 5.0 TB/s).
// Sums are fp64 per 8 elements: the fp32 sum of 8 squares is converted, and
// recomputed in fp64 when it left fp32's range (overflow past 3e38 or below
// 1e-30), which only extreme gradients do.
namespace {

struct NormEntry {
  const void* data;
  long long numel;
  uint32_t first_chunk;
  uint16_t dtype, vec;
};
template <int N>
struct NormArgs {
  double* partial;
  uint32_t n, chunks;
  NormEntry e[N];
};
constexpr int kNormLoads = 8;  // of a thread, in flight together
constexpr int kNormChunk = kThreads * 8 * kNormLoads;
constexpr int kNormLarge = 1300;
static_assert(sizeof(NormArgs<kNormLarge>) <= 32764, "kernel arguments");
constexpr unsigned kNormCtas = 148 * 8;  // one wave of eight 256-thread CTAs per SM

__device__ __forceinline__ double sum_squares(const float (&v)[8]) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += v[j] * v[j];
  if (s > 1e-30f && s <= 3.402823466e38f) return (double)s;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) d += (double)v[j] * (double)v[j];
  return d;
}

template <typename T>
__device__ __forceinline__ double norm_chunk(const NormEntry& t, long long start) {
  const T* p = static_cast<const T*>(t.data);
  double acc = 0.0;
  if (t.vec && start + kNormChunk <= t.numel) {
    constexpr int kHalf = kNormLoads / ((int)sizeof(T) / 2);  // fp32: 16-byte loads twice as many
    Raw8<T> r[kHalf];
#pragma unroll
    for (int k = 0; k < kNormLoads; k += kHalf) {
#pragma unroll
      for (int i = 0; i < kHalf; ++i) r[i].load(p + start + ((k + i) * kThreads + threadIdx.x) * 8);
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        float v[8];
        r[i].get(v);
        acc += sum_squares(v);
      }
    }
    return acc;
  }
#pragma unroll 1
  for (int i = 0; i < kNormLoads; ++i) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long k = start + (i * 8 + j) * kThreads + threadIdx.x;
      v[j] = k < t.numel ? to_f<T>(p[k]) : 0.0f;
    }
    acc += sum_squares(v);
  }
  return acc;
}

// Sum over the CTA, in a fixed order; the result is thread 0's.
__device__ __forceinline__ double cta_sum(double x) {
  __shared__ double s[kWarps];
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
  __syncthreads();
  double r = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < kWarps; ++w) r += s[w];
  return r;
}

template <int N>
__global__ void __launch_bounds__(kThreads) grad_norm_partial_kernel(const __grid_constant__ NormArgs<N> a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    uint32_t lo = 0, hi = a.n - 1;
    while (lo < hi) {
      const uint32_t mid = (lo + hi + 1) >> 1;
      if (a.e[mid].first_chunk <= c) lo = mid;
      else hi = mid - 1;
    }
    const NormEntry& t = a.e[lo];
    const long long start = (long long)(c - t.first_chunk) * kNormChunk;
    if (t.dtype == DCN_FLOAT32) acc += norm_chunk<float>(t, start);
    else if (t.dtype == DCN_FLOAT16) acc += norm_chunk<__half>(t, start);
    else acc += norm_chunk<__nv_bfloat16>(t, start);
  }
  const double r = cta_sum(acc);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = r;
}

__global__ void __launch_bounds__(kThreads) grad_norm_finish_kernel(const double* partial, unsigned n, double max_norm,
                                                                    double loss_scale, float* norm, float* factor) {
  // launched beside the partial sums; waits for them here
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double acc = 0.0;
  for (unsigned i = threadIdx.x; i < n; i += kThreads) acc += partial[i];
  const double s = cta_sum(acc);
  if (threadIdx.x != 0) return;
  const double total = sqrt(s) / loss_scale;
  *norm = (float)total;
  // not finite (as fp32 holds it): NaN, which makes the optimizer step skip itself
  const bool finite = fabsf((float)total) <= 3.402823466e38f;
  const double clip = max_norm < 0.0 ? 1.0 : fmin(1.0, max_norm / (total + 1e-6));
  *factor = finite ? (float)(clip / loss_scale) : __int_as_float(0x7fffffff);
}

template <int N>
cudaError_t norm_launch(const NormEntry* e, uint32_t n, uint32_t chunks, unsigned ctas, double* partial,
                        cudaStream_t st) {
  NormArgs<N> a;
  a.partial = partial;
  a.n = n;
  a.chunks = chunks;
  std::copy(e, e + n, a.e);
  KernelScope ks("grad_norm_partial", st);
  grad_norm_partial_kernel<N><<<ctas, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

// The launches of a call: [first tensor, tensor count, chunks, CTAs].
struct NormPart {
  int64_t first, count;
  unsigned long long chunks;
  unsigned ctas;
};
std::vector<NormPart> norm_parts(const dcn_tensor_ref* t, int64_t n) {
  std::vector<NormPart> parts;
  int64_t i = 0;
  while (i < n) {
    NormPart p{i, 0, 0, 0};
    while (i < n && p.count < kNormLarge) {
      const unsigned long long c = ((unsigned long long)t[i].numel + kNormChunk - 1) / kNormChunk;
      if (p.count && p.chunks + c > 0x7fffffffull) break;
      p.chunks += c;
      ++p.count;
      ++i;
    }
    p.ctas = (unsigned)std::min<unsigned long long>(p.chunks, kNormCtas);
    parts.push_back(p);
  }
  return parts;
}

}  // namespace

size_t grad_norm_workspace(const dcn_tensor_ref* t, int64_t n) {
  size_t ctas = 0;
  for (const NormPart& p : norm_parts(t, n)) ctas += p.ctas;
  return ws_align(sizeof(double) * std::max<size_t>(ctas, 1));
}

cudaError_t grad_norm(const dcn_tensor_ref* t, int64_t n, double max_norm, double loss_scale, float* norm,
                      float* factor, void* workspace, cudaStream_t st) {
  double* partial = static_cast<double*>(workspace);
  unsigned used = 0;
  for (const NormPart& p : norm_parts(t, n)) {
    if (!p.ctas) continue;
    std::vector<NormEntry> e((size_t)p.count);
    uint32_t chunk = 0;
    for (int64_t k = 0; k < p.count; ++k) {
      const dcn_tensor_ref& r = t[p.first + k];
      e[k] = {r.data, r.numel, chunk, (uint16_t)r.dtype, (uint16_t)aligned(r.data, 16)};
      chunk += (uint32_t)((r.numel + kNormChunk - 1) / kNormChunk);
    }
    auto go = [&](auto cap) {
      return norm_launch<decltype(cap)::value>(e.data(), (uint32_t)p.count, chunk, p.ctas, partial + used, st);
    };
    const cudaError_t err = p.count <= 32    ? go(std::integral_constant<int, 32>{})
                            : p.count <= 160 ? go(std::integral_constant<int, 160>{})
                                             : go(std::integral_constant<int, kNormLarge>{});
    if (err != cudaSuccess) return err;
    used += p.ctas;
  }
  KernelScope ks("grad_norm_finish", st);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = used ? 1 : 0;  // no partial sums: nothing to overlap with
  return cudaLaunchKernelEx(&cfg, grad_norm_finish_kernel, (const double*)partial, used, max_norm, loss_scale, norm, factor);
}

}  // namespace dcn
