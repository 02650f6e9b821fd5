// AdamW step over many tensors:
//   m = b1 m + (1-b1) g,  v = b2 v + (1-b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// The bound is HBM: 28 bytes an element for f32 parameters and states, 16 and
// a bit with 8-bit states.  One launch covers up to 256 tensors, whose
// descriptors travel as kernel parameters (no copy to the device, nothing to
// keep between calls).  CTAs are persistent: the step's scalars (two powers in
// double) are formed once, and each CTA goes over chunks of 2048 elements of
// one tensor.  A warp owns blocks of 256 elements, 8 a lane in two groups of 4
// neighbours, so f32 data moves in coalesced 16-byte accesses and an 8-bit
// state's scale is one warp reduction.
//
// The states' sums are made in the order written above with every operation
// rounded (the file is compiled without multiply-add contraction), so they are
// the same as the elementary f32 operations one after the other; p's quotient
// is a product with an approximate reciprocal, 2^-22 of the step.  8-bit states
// hold m and sqrt(v) as e4m3 (4 significant bits, 2^-9 .. 448) of the value
// over its block's largest.  Their rounding is random, up with the
// probability of the remainder: with b2 = 0.999 a step changes v by about
// 0.1 %, nearest rounding to a code 6 % away would never move it.  A NaN keeps its
// element's codes NaN and is left out of the block's largest value; an infinite
// one makes its scale infinite, and the block NaN at the next step.  The bits
// come from the lowbias32 mixer (C. Wellons, "Prospecting for Hash
// Functions") of element, tensor and step.
//
// Measured: 302 M elements, bf16 parameters and gradients, f32 masters and
// states: 1.38 ms, 6.1 TB/s.  151 M f32 elements with 8-bit states: 0.53 ms,
// 4.6 TB/s; there neither issue slots (69 % taken) nor DRAM (55 %) are full: a
// warp loads, codes and stores a chunk before it loads the next, so memory and
// the instructions of rounding and coding wait for one another.
#include <cuda_fp8.h>

#include "amc_half.cuh"
#include "amc_internal.h"
#include "amc_tc.cuh"

namespace amc {

using tc::add2;
using tc::max3;
using tc::min3_nan;
using tc::mul2;

namespace {

constexpr int kAdamTensors = 256;    // descriptors per launch
constexpr int kAdamChunk = 2048;     // elements of a CTA's pass: a block a warp
constexpr int64_t kAdamMost = (int64_t)0x7fffffff * kAdamChunk;
constexpr int kAdamCtas = 4;         // a SM, at 64 registers a thread
constexpr int kAdamBlock = 256;      // elements per scale
constexpr float kE4m3Max = 448.f;
constexpr uint32_t kE4m3Nan = 127;

struct AdamTensor {
  amc_adamw_tensor t;
  int64_t chunk0;     // its first chunk
};

struct AdamArgs {
  int64_t* state;
  const float* lr_dev;
  double lr, b1, b2;
  float eps;
  double wd;
  int64_t chunks;
  int count, base, last;   // tensors here, index of the first, whether this launch ends the step
  AdamTensor t[kAdamTensors];
};
static_assert(sizeof(AdamArgs) <= 32764, "kernel parameters");

__device__ __forceinline__ double int_pow(double x, int64_t n) {
  double r = 1.0;
  for (; n > 0; n >>= 1) {
    if (n & 1) r *= x;
    x *= x;
  }
  return r;
}

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  return x ^ (x >> 16);
}

// A value in [0, 448] (a hair above from rounding) to its 7-bit e4m3 code with
// 20 random bits.  From 2^-6 up the bits are added below the third bit of the
// mantissa and cut off; below, the codes are steps of 2^-9, and
// floor(512 a + bits 2^-20) comes out of the low bits of a sum with 2^23 that
// is rounded down.  No conversion instruction (16 a clock) is needed.
constexpr float kE4m3Fine = 0.015625f;
__device__ __forceinline__ uint32_t e4m3_coarse(uint32_t bits, uint32_t rnd) {
  return min(((bits + rnd) >> 20) - (120u << 3), 126u);
}
__device__ __forceinline__ uint32_t e4m3_fine(float a, uint32_t rnd) {
  const float part = __uint_as_float(0x3F800000u | rnd << 3) - 1.f;   // rnd 2^-20
  return __float_as_uint(__fadd_rd(a * 512.f + part, 8388608.f)) & 15u;
}
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 get2(const float (&v)[4], int k) { return make_float2(v[k], v[k + 1]); }
__device__ __forceinline__ void put2(float (&v)[4], int k, float2 x) {
  v[k] = x.x;
  v[k + 1] = x.y;
}
// Four codes to their values (the 8-bit pairs convert through fp16, which holds them exactly).
__device__ __forceinline__ void e4m3_values(float (&v)[4], uint32_t w) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * k) & 0xFFFFu), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}

// 4 neighbours, as one access where the block is whole and aligned.
template <typename T>
__device__ __forceinline__ void load4(float (&v)[4], const T* p, int64_t e, int64_t n, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + e);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(p + e);
      const float2 a = unpack2<T>(x.x), b = unpack2<T>(x.y);
      v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = e + k < n ? to_f32(p[e + k]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4], int64_t e, int64_t n, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p + e) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>(p + e) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (e + k < n) p[e + k] = from_f32<T>(v[k]);
  }
}
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int64_t e, int64_t n, bool vec) {
  if (vec) return *reinterpret_cast<const uint32_t*>(p + e);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (e + k < n) w |= (uint32_t)p[e + k] << (8 * k);
  return w;
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint32_t w, int64_t e, int64_t n, bool vec) {
  if (vec) {
    *reinterpret_cast<uint32_t*>(p + e) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (e + k < n) p[e + k] = (uint8_t)(w >> (8 * k));
  }
}
// A sum of two products, each rounded: written as a packed sum, the assembler
// contracts it with one of them.
__device__ __forceinline__ float2 sum2(float2 a, float2 b) {
  return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y));
}
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

}  // namespace

template <typename P, typename G, bool MASTER, bool BITS8>
__global__ void __launch_bounds__(256, kAdamCtas) k_adamw(const __grid_constant__ AdamArgs a) {
  __shared__ float sh[3];
  __shared__ uint32_t sh_t;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    const int64_t step = a.state[0] + 1;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    sh[0] = (float)(lr / (1.0 - int_pow(a.b1, step)));
    sh[1] = (float)(1.0 / sqrt(1.0 - int_pow(a.b2, step)));
    sh[2] = (float)(1.0 - lr * a.wd);
    sh_t = (uint32_t)step;
  }
  const float b1 = (float)a.b1, b2 = (float)a.b2, r1 = (float)(1.0 - a.b1), r2 = (float)(1.0 - a.b2);
  __syncthreads();
  const float rate = sh[0], root = sh[1], keep = sh[2];
  int lo = 0;
  for (int64_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    // the last tensor that starts at or before this chunk, by bisection of those still ahead
    int hi = a.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.t[mid].chunk0 <= chunk) lo = mid;
      else hi = mid - 1;
    }
    const amc_adamw_tensor& t = a.t[lo].t;
    const int64_t n = t.n, e0 = (chunk - a.t[lo].chunk0) * kAdamChunk + warp * kAdamBlock;
    if (e0 >= n) continue;
    // aligned for 4-element accesses of every array (blocks start on multiples of 256)
    const uintptr_t al = (uintptr_t)t.m | (uintptr_t)t.v;
    bool vec = e0 + kAdamBlock <= n && !(al & (BITS8 ? 3 : 15)) && !((uintptr_t)t.p & (4 * sizeof(P) - 1)) &&
               !((uintptr_t)t.g & (4 * sizeof(G) - 1));
    if (MASTER) vec = vec && !((uintptr_t)t.master & 15);
    const uint32_t seed = sh_t * 0x85EBCA77u + (uint32_t)(a.base + lo) * 0xC2B2AE3Du;
    float p[2][4], g[2][4], m[2][4], v[2][4];
    uint32_t cm[2], cv[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t e = e0 + 128 * j + 4 * lane;
      if (MASTER) load4(p[j], t.master, e, n, vec);
      else load4(p[j], (const P*)t.p, e, n, vec);
      load4(g[j], (const G*)t.g, e, n, vec);
      if (BITS8) {
        cm[j] = load_codes((const uint8_t*)t.m, e, n, vec);
        cv[j] = load_codes((const uint8_t*)t.v, e, n, vec);
      } else {
        load4(m[j], (const float*)t.m, e, n, vec);
        load4(v[j], (const float*)t.v, e, n, vec);
      }
    }
    if (BITS8) {
      const float sm = t.m_scale[e0 / kAdamBlock], sv = t.v_scale[e0 / kAdamBlock];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        e4m3_values(m[j], cm[j]);
        e4m3_values(v[j], cv[j]);
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          put2(m[j], k, mul2(get2(m[j], k), twice(sm)));
          const float2 u = mul2(get2(v[j], k), twice(sv));
          put2(v[j], k, mul2(u, u));
        }
      }
    }
    float top_m = 0.f, top_u = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        const float2 gg = get2(g[j], k);
        const float2 mm = sum2(mul2(get2(m[j], k), twice(b1)), mul2(gg, twice(r1)));
        const float2 vv = sum2(mul2(get2(v[j], k), twice(b2)), mul2(mul2(gg, gg), twice(r2)));
        const float2 u = make_float2(__fsqrt_rn(vv.x), __fsqrt_rn(vv.y));
        const float2 den = add2(mul2(u, twice(root)), twice(a.eps));
        const float2 step = mul2(mm, make_float2(reciprocal(den.x), reciprocal(den.y)));
        put2(p[j], k, add2(mul2(get2(p[j], k), twice(keep)), mul2(twice(-rate), step)));
        put2(m[j], k, mm);
        put2(v[j], k, BITS8 ? u : vv);
        if (BITS8) {
          top_m = max3(top_m, fabsf(mm.x), fabsf(mm.y));
          top_u = max3(top_u, u.x, u.y);
        }
      }
    if (BITS8) {
      top_m = warp_max(top_m);
      top_u = warp_max(top_u);
      const bool some_m = top_m >= 7.888609052210118e-31f, some_u = top_u >= 7.888609052210118e-31f;   // 2^-100
      const float im = some_m ? 1.f / top_m * kE4m3Max : 0.f, iu = some_u ? 1.f / top_u * kE4m3Max : 0.f;
      if (lane == 0) {
        t.m_scale[e0 / kAdamBlock] = some_m ? top_m * (1.f / kE4m3Max) : 0.f;
        t.v_scale[e0 / kAdamBlock] = some_u ? top_u * (1.f / kE4m3Max) : 0.f;
      }
      // values over their scale; m keeps its sign
      float least = 448.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const float2 x = mul2(get2(m[j], k), twice(im)), u = mul2(get2(v[j], k), twice(iu));
          put2(m[j], k, x);
          put2(v[j], k, u);
          least = min3_nan(least, fabsf(x.x), fabsf(x.y));
          least = min3_nan(least, u.x, u.y);
        }
      // below 2^-6 of 448 the codes are even steps: about one block in forty
      // of normally distributed values has any, and takes the longer way, as
      // one that holds NaN does
      const bool fine = __any_sync(0xffffffffu, !(least >= kE4m3Fine));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t x = (uint32_t)(e0 + 128 * j + 4 * lane) * 0x9E3779B1u + seed;
        cm[j] = cv[j] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k, x += 0x9E3779B1u) {
          const uint32_t rnd = mix32(x), bits = __float_as_uint(m[j][k]);
          uint32_t c = e4m3_coarse(bits & 0x7FFFFFFFu, rnd & 0xFFFFFu), d = e4m3_coarse(__float_as_uint(v[j][k]), rnd >> 12);
          if (fine) {
            if (fabsf(m[j][k]) < kE4m3Fine) c = e4m3_fine(fabsf(m[j][k]), rnd & 0xFFFFFu);
            if (v[j][k] < kE4m3Fine) d = max(e4m3_fine(v[j][k], rnd >> 12), v[j][k] > 0.f ? 1u : 0u);
            if (isnan(m[j][k])) c = kE4m3Nan;
            if (isnan(v[j][k])) d = kE4m3Nan;
          }
          cm[j] |= (c | bits >> 31 << 7) << (8 * k);
          cv[j] |= d << (8 * k);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t e = e0 + 128 * j + 4 * lane;
      if (MASTER) store4(t.master, p[j], e, n, vec);
      store4((P*)t.p, p[j], e, n, vec);
      if (BITS8) {
        store_codes((uint8_t*)t.m, cm[j], e, n, vec);
        store_codes((uint8_t*)t.v, cv[j], e, n, vec);
      } else {
        store4((float*)t.m, m[j], e, n, vec);
        store4((float*)t.v, v[j], e, n, vec);
      }
    }
  }
  if (a.last && threadIdx.x == 0) {
    // the last CTA of the step counts it; every CTA has read the old count
    __threadfence();
    if (atomicAdd((unsigned long long*)&a.state[1], 1ull) == gridDim.x - 1) {
      a.state[0] += 1;
      a.state[1] = 0;
    }
  }
}

namespace {

template <typename P, typename G>
int adamw_launch(const AdamArgs& a, unsigned grid, bool master, bool bits8, cudaStream_t s) {
  if (master && bits8) k_adamw<P, G, true, true><<<grid, 256, 0, s>>>(a);
  else if (master) k_adamw<P, G, true, false><<<grid, 256, 0, s>>>(a);
  else if (bits8) k_adamw<P, G, false, true><<<grid, 256, 0, s>>>(a);
  else k_adamw<P, G, false, false><<<grid, 256, 0, s>>>(a);
  AMC_CUDA(cudaGetLastError());
  return AMC_OK;
}

template <typename P>
int adamw_grad(const AdamArgs& a, int32_t g_dtype, unsigned grid, bool master, bool bits8, cudaStream_t s) {
  if (g_dtype == AMC_F32) return adamw_launch<P, float>(a, grid, master, bits8, s);
  if (g_dtype == AMC_BF16) return adamw_launch<P, __nv_bfloat16>(a, grid, master, bits8, s);
  return adamw_launch<P, __half>(a, grid, master, bits8, s);
}

bool layer_dtype(int32_t d) { return d == AMC_F32 || d == AMC_BF16 || d == AMC_F16; }

}  // namespace

}  // namespace amc

using namespace amc;

extern "C" {

int amc_adamw(const amc_adamw_tensor* t, int32_t count, int32_t p_dtype, int32_t g_dtype, int32_t state_dtype,
              int64_t* step_state, const float* lr_dev, double lr, double beta1, double beta2, double eps,
              double weight_decay, void* stream) {
  if (count < 0 || (count && !t) || !step_state) return fail(AMC_ERR_INVALID, "amc_adamw: null argument");
  if (!layer_dtype(p_dtype) || !layer_dtype(g_dtype) || (state_dtype != AMC_F32 && state_dtype != AMC_E4M3))
    return fail(AMC_ERR_INVALID, "amc_adamw: parameters and gradients f32, bf16 or f16; states f32 or e4m3");
  if (!(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(weight_decay >= 0) || !(lr >= 0))
    return fail(AMC_ERR_INVALID, "amc_adamw: betas in [0, 1), lr, eps and weight_decay not negative");
  const bool bits8 = state_dtype == AMC_E4M3;
  bool master = false;
  int64_t all = 0;
  for (int i = 0; i < count && !master; ++i) master = t[i].n > 0 && t[i].master;
  for (int i = 0; i < count; ++i) {
    const amc_adamw_tensor& x = t[i];
    if (x.n < 0) return fail(AMC_ERR_INVALID, "amc_adamw: negative size");
    // chunks are counted in 32 bits, and no launch is made of a step that fails
    if (x.n > kAdamMost || (all += x.n / kAdamChunk + 1) > 0x7fffffff)
      return fail(AMC_ERR_INVALID, "amc_adamw: too many elements");
    if (x.n && (!x.p || !x.g || !x.m || !x.v)) return fail(AMC_ERR_INVALID, "amc_adamw: null tensor");
    if (x.n && (x.master != nullptr) != master) return fail(AMC_ERR_INVALID, "amc_adamw: masters for all tensors or for none");
    if (x.n && bits8 && (!x.m_scale || !x.v_scale)) return fail(AMC_ERR_INVALID, "amc_adamw: 8-bit states need their scales");
  }
  if (fault_injected("launch")) return fail(AMC_ERR_INJECTED, "adamw: injected launch failure (AMC_FAULT=launch)");
  cudaStream_t s = pick_stream(stream);
  AdamArgs a;
  a.state = step_state;
  a.lr_dev = lr_dev;
  a.lr = lr;
  a.b1 = beta1;
  a.b2 = beta2;
  a.eps = (float)eps;
  a.wd = weight_decay;
  int i = 0;
  do {
    a.base = i;
    a.count = 0;
    int64_t chunks = 0;
    for (; i < count && a.count < kAdamTensors; ++i) {
      a.t[a.count].t = t[i];
      a.t[a.count++].chunk0 = chunks;
      chunks += (t[i].n + kAdamChunk - 1) / kAdamChunk;
    }
    a.last = i == count;
    if (!a.count) {   // no tensor: an empty one still counts the step
      a.t[0] = AdamTensor{};
      a.count = 1;
    }
    if (!chunks && !a.last) continue;
    a.chunks = chunks;
    const int64_t most = (int64_t)num_sms() * kAdamCtas;
    const unsigned grid = (unsigned)(chunks < 1 ? 1 : chunks < most ? chunks : most);
    int rc = p_dtype == AMC_F32    ? adamw_grad<float>(a, g_dtype, grid, master, bits8, s)
             : p_dtype == AMC_BF16 ? adamw_grad<__nv_bfloat16>(a, g_dtype, grid, master, bits8, s)
                                   : adamw_grad<__half>(a, g_dtype, grid, master, bits8, s);
    if (rc) return rc;
  } while (i < count);
  return AMC_OK;
}

}  // extern "C"
