// Rotary positions: pair i of a row at position p turns by p * freqs[i].
//   a' = ms (a cos - b sin),  b' = ms (b cos + a sin);  the inverse turn is
//   the gradient (the transpose of the same matrix).
// The bound is HBM: each element is read and written once.  A thread keeps
// the sines of V pairs of one row in registers and applies them to every head
// of that row it owns, so the angles cost little: the turn count is formed
// and reduced to half a turn in f64 (a position of 2^40 keeps its angle), its
// sine and cosine in f32.  No table is read.
#include <cmath>

#include "amc_half.cuh"
#include "amc_internal.h"

namespace amc {

namespace {

constexpr int kRopeThreads = 256;

struct RopeArgs {
  amc_rope_tensor t[2];
  int chunks0;                 // head chunks of tensor 0; the rest are tensor 1's
  int heads_per;               // heads per chunk
  int64_t rows, n;             // batch * n, n
  int d, rot, pair_units, units;
  const int64_t* pos;
  int64_t pos_stride;
  const double* freqs;
  float mscale;
  int inverse;
};

template <typename T, int V>
struct Vec {
  static constexpr int bytes = V * (int)sizeof(T);
  T e[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (bytes == 32) {
      reinterpret_cast<int4*>(e)[0] = reinterpret_cast<const int4*>(p)[0];
      reinterpret_cast<int4*>(e)[1] = reinterpret_cast<const int4*>(p)[1];
    } else if constexpr (bytes == 16) {
      *reinterpret_cast<int4*>(e) = *reinterpret_cast<const int4*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (bytes == 32) {
      reinterpret_cast<int4*>(p)[0] = reinterpret_cast<const int4*>(e)[0];
      reinterpret_cast<int4*>(p)[1] = reinterpret_cast<const int4*>(e)[1];
    } else if constexpr (bytes == 16) {
      *reinterpret_cast<int4*>(p) = *reinterpret_cast<const int4*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = e[i];
    }
  }
};

}  // namespace

// One thread: one row, V pairs (or V copied elements behind rot), heads_per heads.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) k_rope(const __grid_constant__ RopeArgs a) {
  const int64_t id = (int64_t)blockIdx.x * kRopeThreads + threadIdx.x;
  const int64_t row = id / a.units;
  const int u = (int)(id % a.units);
  if (row >= a.rows) return;
  const int which = (int)blockIdx.y >= a.chunks0;
  const amc_rope_tensor& t = a.t[which];
  const int64_t h0 = (int64_t)(blockIdx.y - (which ? a.chunks0 : 0)) * a.heads_per;
  const int64_t h1 = min(h0 + a.heads_per, t.heads);
  const int64_t b = row / a.n, i = row % a.n;
  const T* x = (const T*)t.x + b * t.xs[0] + h0 * t.xs[1] + i * t.xs[2];
  T* o = (T*)t.out + b * t.os[0] + h0 * t.os[1] + i * t.os[2];
  const int64_t xh = t.xs[1], oh = t.os[1];
  if (u >= a.pair_units) {
    const int c = a.rot + (u - a.pair_units) * V;
    for (int64_t h = h0; h < h1; ++h, x += xh, o += oh) {
      Vec<T, V> v;
      v.load(x + c);
      v.store(o + c);
    }
    return;
  }
  float co[V], si[V];
  const double p = (double)a.pos[b * a.pos_stride + i];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    double turns = p * (a.freqs[u * V + k] * 0.15915494309189533577);   // 1 / (2 pi)
    turns -= rint(turns);
    sincospif(2.f * (float)turns, &si[k], &co[k]);
    co[k] *= a.mscale;
    si[k] *= a.inverse ? -a.mscale : a.mscale;
  }
  const int ca = INTER ? u * 2 * V : u * V, cb = INTER ? ca + V : ca + a.rot / 2;
#pragma unroll 4
  for (int64_t h = h0; h < h1; ++h, x += xh, o += oh) {
    Vec<T, V> va, vb;
    va.load(x + ca);
    vb.load(x + cb);
    if constexpr (INTER) {
      float e[2 * V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        e[k] = to_f32(va.e[k]);
        e[V + k] = to_f32(vb.e[k]);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float r = e[2 * k] * co[k] - e[2 * k + 1] * si[k], q = e[2 * k + 1] * co[k] + e[2 * k] * si[k];
        (2 * k < V ? va.e[2 * k < V ? 2 * k : 0] : vb.e[2 * k < V ? 0 : 2 * k - V]) = from_f32<T>(r);
        (2 * k + 1 < V ? va.e[2 * k + 1 < V ? 2 * k + 1 : 0] : vb.e[2 * k + 1 < V ? 0 : 2 * k + 1 - V]) = from_f32<T>(q);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xa = to_f32(va.e[k]), xb = to_f32(vb.e[k]);
        va.e[k] = from_f32<T>(xa * co[k] - xb * si[k]);
        vb.e[k] = from_f32<T>(xb * co[k] + xa * si[k]);
      }
    }
    va.store(o + ca);
    vb.store(o + cb);
  }
}

namespace {

template <typename T, int V>
int rope_launch(RopeArgs& a, int count, bool inter, cudaStream_t s) {
  a.pair_units = a.rot / 2 / V;
  a.units = a.pair_units + (a.d - a.rot) / V;
  const int64_t threads = a.rows * a.units;
  const int64_t blocks = (threads + kRopeThreads - 1) / kRopeThreads;
  if (blocks > 0x7fffffff) return fail(AMC_ERR_INVALID, "amc_rope: too many rows");
  // Heads per thread: as many as leave four full waves of threads.
  const int64_t hmax = count > 1 && a.t[1].heads > a.t[0].heads ? a.t[1].heads : a.t[0].heads;
  int64_t per = 16;
  while (per > 1 && blocks * ((hmax + per - 1) / per) < 4 * (int64_t)num_sms()) per /= 2;
  a.heads_per = (int)per;
  a.chunks0 = (int)((a.t[0].heads + per - 1) / per);
  const int chunks = a.chunks0 + (count > 1 ? (int)((a.t[1].heads + per - 1) / per) : 0);
  const dim3 grid((unsigned)blocks, (unsigned)chunks);
  if (inter) k_rope<T, V, true><<<grid, kRopeThreads, 0, s>>>(a);
  else k_rope<T, V, false><<<grid, kRopeThreads, 0, s>>>(a);
  AMC_CUDA(cudaGetLastError());
  return AMC_OK;
}

// Whether V-element vectors fit every row: pointers, strides and the pair
// and copied ranges are multiples of V elements (16 bytes for V > 1).
template <typename T, int V>
bool rope_fits(const RopeArgs& a, int count) {
  if ((a.rot / 2) % V || (a.d - a.rot) % V) return false;
  for (int k = 0; k < count; ++k) {
    if (((uintptr_t)a.t[k].x | (uintptr_t)a.t[k].out) & 15) return false;
    for (int j = 0; j < 3; ++j)
      if (a.t[k].xs[j] * (int64_t)sizeof(T) % 16 || a.t[k].os[j] * (int64_t)sizeof(T) % 16) return false;
  }
  return true;
}

template <typename T>
int rope_typed(RopeArgs& a, int count, bool inter, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (rope_fits<T, V>(a, count)) return rope_launch<T, V>(a, count, inter, s);
  return rope_launch<T, 1>(a, count, inter, s);
}

}  // namespace

}  // namespace amc

using namespace amc;

extern "C" {

int amc_rope(const amc_rope_tensor* t, int32_t count, int32_t dtype, int64_t batch, int64_t n, int32_t d, int32_t rot,
             const int64_t* pos, int64_t pos_stride, const double* freqs, float mscale, int32_t interleaved,
             int32_t inverse, void* stream) {
  if (!t || count < 1 || count > 2) return fail(AMC_ERR_INVALID, "amc_rope: one or two tensors");
  if (dtype != AMC_F32 && dtype != AMC_BF16 && dtype != AMC_F16)
    return fail(AMC_ERR_INVALID, "amc_rope: dtype must be f32, bf16 or f16");
  if (batch < 0 || n < 0 || d <= 0 || rot <= 0 || rot > d || rot % 2)
    return fail(AMC_ERR_INVALID, "amc_rope: bad sizes (rot even, 2..d)");
  RopeArgs a{};
  bool any = false;
  for (int k = 0; k < count; ++k) {
    a.t[k] = t[k];
    if (t[k].heads < 0 || t[k].heads > 32767) return fail(AMC_ERR_INVALID, "amc_rope: heads 0..32767");
    any = any || t[k].heads > 0;
  }
  if (!any || !batch || !n) return AMC_OK;
  for (int k = 0; k < count; ++k) {
    if (t[k].heads && (!t[k].x || !t[k].out)) return fail(AMC_ERR_INVALID, "amc_rope: null tensor");
    if (t[k].x == t[k].out)
      for (int j = 0; j < 3; ++j)
        if (t[k].xs[j] != t[k].os[j]) return fail(AMC_ERR_INVALID, "amc_rope: in place needs the same strides");
  }
  if (!pos || !freqs) return fail(AMC_ERR_INVALID, "amc_rope: null positions or frequencies");
  if (n > ((int64_t)1 << 40) / batch) return fail(AMC_ERR_INVALID, "amc_rope: too many rows");
  if (fault_injected("launch")) return fail(AMC_ERR_INJECTED, "rope: injected launch failure (AMC_FAULT=launch)");
  a.rows = batch * n;
  a.n = n;
  a.d = d;
  a.rot = rot;
  a.pos = pos;
  a.pos_stride = pos_stride;
  a.freqs = freqs;
  a.mscale = mscale;
  a.inverse = inverse;
  cudaStream_t s = pick_stream(stream);
  if (dtype == AMC_F32) return rope_typed<float>(a, count, interleaved != 0, s);
  if (dtype == AMC_BF16) return rope_typed<__nv_bfloat16>(a, count, interleaved != 0, s);
  return rope_typed<__half>(a, count, interleaved != 0, s);
}

int amc_rope_freqs(double* out, int32_t rot, double base, int32_t kind, double factor, int64_t original_len,
                   double slow, double fast, float* mscale) {
  if (!out || !mscale || rot <= 0 || rot % 2) return fail(AMC_ERR_INVALID, "amc_rope_freqs: rot even and positive");
  if (!(base > 0) || !(factor > 0) || kind < AMC_ROPE_PLAIN || kind > AMC_ROPE_PARTS)
    return fail(AMC_ERR_INVALID, "amc_rope_freqs: bad base, factor or kind");
  if (kind == AMC_ROPE_PARTS && (original_len <= 0 || !(fast > slow)))
    return fail(AMC_ERR_INVALID, "amc_rope_freqs: original_len > 0 and fast > slow expected");
  if (kind == AMC_ROPE_BASE) {
    if (rot < 4) return fail(AMC_ERR_INVALID, "amc_rope_freqs: a raised base needs rot of 4 or more");
    base *= pow(factor, (double)rot / (rot - 2));
  }
  for (int i = 0; i < rot / 2; ++i) {
    double f = pow(base, -2.0 * i / rot);
    if (kind == AMC_ROPE_LINEAR) f /= factor;
    if (kind == AMC_ROPE_PARTS) {
      const double turns = (double)original_len * f * 0.15915494309189533577;
      double keep = (turns - slow) / (fast - slow);
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      f = f * keep + f / factor * (1 - keep);
    }
    out[i] = f;
  }
  *mscale = kind == AMC_ROPE_PARTS && factor > 1 ? (float)(0.1 * log(factor) + 1.0) : 1.f;
  return AMC_OK;
}

}  // extern "C"
