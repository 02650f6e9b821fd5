// AdamW step over many tensors:
//   m = b1 m + (1-b1) g,  v = b2 v + (1-b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// The bound is HBM: 28 bytes an element for f32 parameters and states, 16 and
// a bit with 8-bit states.  One launch covers up to 256 tensors, whose
// descriptors travel as kernel parameters (no copy to the device, nothing to
// keep between calls); a CTA owns 4096 elements of one tensor and finds it by
// bisection.  A warp owns blocks of 256 elements, 8 a lane in two groups of 4
// neighbours, so f32 data moves in coalesced 16-byte accesses and an 8-bit
// state's scale is one warp reduction.
//
// The sums are made in the order written above with every operation rounded
// (the file is compiled without multiply-add contraction), so the step is the
// same as the elementary f32 operations one after the other.  8-bit states
// hold m and sqrt(v) as e4m3 (4 significant bits, 2^-9 .. 448) of the value
// over its block's largest.  Their rounding is random, up with the
// probability of the remainder: with b2 = 0.999 a step changes v by about
// 0.1 %, nearest rounding to a code 6 % away would never move it.  The bits
// come from the lowbias32 mixer (C. Wellons, "Prospecting for Hash
// Functions") of element, tensor and step.
#include "amc_half.cuh"
#include "amc_internal.h"

namespace amc {

namespace {

constexpr int kAdamTensors = 256;    // descriptors per launch
constexpr int kAdamChunk = 4096;     // elements per CTA
constexpr int kAdamBlock = 256;      // elements per scale
constexpr float kE4m3Max = 448.f;

struct AdamTensor {
  amc_adamw_tensor t;
  int64_t chunk0;     // first CTA of this tensor
};

struct AdamArgs {
  int64_t* state;
  const float* lr_dev;
  double lr, b1, b2;
  float eps;
  double wd;
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

// a in [0, 448] (a hair above from rounding): to e4m3 with 20 random bits.
// Returns the 7-bit code.
__device__ __forceinline__ uint32_t e4m3_random(float a, uint32_t rnd) {
  if (a < 0.015625f) return (uint32_t)floorf(a * 512.f + (float)rnd * 9.5367431640625e-07f);   // steps of 2^-9
  const uint32_t c = ((__float_as_uint(a) + rnd) >> 20) - (120u << 3);
  return c > 126u ? 126u : c;
}
__device__ __forceinline__ float e4m3_value(uint32_t c) {
  const uint32_t m = c & 127u;
  const float v = m < 8u ? (float)m * 0.001953125f : __uint_as_float((m + (120u << 3)) << 20);
  return c & 128u ? -v : v;
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
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

}  // namespace

template <typename P, typename G, bool MASTER, bool BITS8>
__global__ void __launch_bounds__(256) k_adamw(const __grid_constant__ AdamArgs a) {
  __shared__ float sh[3];
  __shared__ uint32_t sh_t;
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].chunk0 <= (int64_t)blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const amc_adamw_tensor& t = a.t[lo].t;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = t.n, c0 = ((int64_t)blockIdx.x - a.t[lo].chunk0) * kAdamChunk;
  if (threadIdx.x == 0) {
    const int64_t step = a.state[0] + 1;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    sh[0] = (float)(lr / (1.0 - int_pow(a.b1, step)));
    sh[1] = (float)sqrt(1.0 - int_pow(a.b2, step));
    sh[2] = (float)(1.0 - lr * a.wd);
    sh_t = (uint32_t)step;
  }
  // aligned for 4-element accesses of every array (chunks start on multiples of 4096)
  const uintptr_t al = (uintptr_t)t.m | (uintptr_t)t.v;
  bool aligned = !(al & (BITS8 ? 3 : 15)) && !((uintptr_t)t.p & (4 * sizeof(P) - 1)) && !((uintptr_t)t.g & (4 * sizeof(G) - 1));
  if (MASTER) aligned = aligned && !((uintptr_t)t.master & 15);
  const float b1 = (float)a.b1, b2 = (float)a.b2, r1 = (float)(1.0 - a.b1), r2 = (float)(1.0 - a.b2);
  __syncthreads();
  const float rate = sh[0], root = sh[1], keep = sh[2];
  const uint32_t seed = sh_t * 0x85EBCA77u + (uint32_t)(a.base + lo) * 0xC2B2AE3Du;
#pragma unroll
  for (int r = 0; r < kAdamChunk / (8 * kAdamBlock); ++r) {
    const int64_t e0 = c0 + (r * 8 + warp) * kAdamBlock;
    if (e0 >= n) continue;
    const bool vec = aligned && e0 + kAdamBlock <= n;
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
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          m[j][k] = e4m3_value(cm[j] >> (8 * k) & 255u) * sm;
          const float u = e4m3_value(cv[j] >> (8 * k) & 255u) * sv;
          v[j][k] = u * u;
        }
    }
    float top_m = 0.f, top_u = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[j][k] = m[j][k] * b1 + g[j][k] * r1;
        v[j][k] = v[j][k] * b2 + (g[j][k] * g[j][k]) * r2;
        const float u = sqrtf(v[j][k]);
        p[j][k] = p[j][k] * keep - rate * (m[j][k] / (u / root + a.eps));
        if (BITS8) {
          v[j][k] = u;
          top_m = fmaxf(top_m, fabsf(m[j][k]));
          top_u = fmaxf(top_u, u);
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
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        cm[j] = cv[j] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t rnd = mix32((uint32_t)(e0 + 128 * j + 4 * lane + k) * 0x9E3779B1u + seed);
          const uint32_t neg = __float_as_uint(m[j][k]) >> 31 << 7;
          cm[j] |= (e4m3_random(fabsf(m[j][k]) * im, rnd & 0xFFFFFu) | neg) << (8 * k);
          const float u = v[j][k] * iu;
          uint32_t c = e4m3_random(u, rnd >> 12);
          if (c == 0 && u > 0.f) c = 1;
          cv[j] |= c << (8 * k);
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
  for (int i = 0; i < count && !master; ++i) master = t[i].n > 0 && t[i].master;
  for (int i = 0; i < count; ++i) {
    const amc_adamw_tensor& x = t[i];
    if (x.n < 0) return fail(AMC_ERR_INVALID, "amc_adamw: negative size");
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
    if (chunks > 0x7fffffff) return fail(AMC_ERR_INVALID, "amc_adamw: too many elements");
    if (!chunks && !a.last) continue;
    const unsigned grid = chunks ? (unsigned)chunks : 1u;
    int rc = p_dtype == AMC_F32    ? adamw_grad<float>(a, g_dtype, grid, master, bits8, s)
             : p_dtype == AMC_BF16 ? adamw_grad<__nv_bfloat16>(a, g_dtype, grid, master, bits8, s)
                                   : adamw_grad<__half>(a, g_dtype, grid, master, bits8, s);
    if (rc) return rc;
  } while (i < count);
  return AMC_OK;
}

}  // extern "C"
