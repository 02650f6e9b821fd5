// Rotary positions: pair i of a row at position p turns by p * freqs[i].
//   a' = ms (a cos - b sin),  b' = ms (b cos + a sin);  the inverse turn is
//   the gradient (the transpose of the same matrix).
// The bound is HBM: each element is read and written once.  A warp owns one row
// (a position) of the batch: its lanes form the sines and cosines of the row's
// pairs once, into shared memory, and then go over the 16-byte vectors of every
// head of both tensors, four in flight a lane, so a position's heads, which a
// projection leaves side by side, move in whole lines.  The first vectors are
// loaded before the angles are formed.  The turn count is a product of two-part
// doubles: a single one, off by 2^-52 of itself, is right to f32's last bits up to
// positions of about 2^30 only, this one up to the 2^53 that a double counts.  What
// is left of it after whole turns goes to f32 for sine and cosine.  No table is
// read.
// Measured: queries and keys of 16 x 2048 tokens, 16 heads each, d 64, bf16
// (268 MB): 46 us, 5.8 TB/s; 16 tokens: 2.8 us in a graph, a launch.
#include <cmath>

#include "amc_half.cuh"
#include "amc_internal.h"

namespace amc {

namespace {

constexpr int kRopeWarps = 4;
constexpr int kRopeFlight = 4;       // vectors (pairs of them) in flight a lane
constexpr int kRopeMaxRot = 1024;
constexpr double kTurn = 0.15915494309189535, kTurnLow = -9.839338337591243e-18;   // 1 / (2 pi) and the rest of it

struct RopeArgs {
  amc_rope_tensor t[2];
  int64_t rows, n;             // batch * n, n
  int d, rot, pair_units, units;   // V pairs each, and with the V-element pieces behind rot
  int items0, items;           // vectors of a row: of tensor 0, of both
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
    if constexpr (bytes == 16) {
      *reinterpret_cast<int4*>(e) = *reinterpret_cast<const int4*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (bytes == 16) {
      *reinterpret_cast<int4*>(p) = *reinterpret_cast<const int4*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = e[i];
    }
  }
};

}  // namespace

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRopeWarps * 32) k_rope(const __grid_constant__ RopeArgs a) {
  extern __shared__ float2 rope_sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kRopeWarps + warp;
  if (row >= a.rows) return;
  float2* turn = rope_sm + warp * (a.rot / 2);   // (cos, sin) of each pair
  const int64_t b = row / a.n, i = row % a.n;
  const T* x[2];
  T* o[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    x[k] = (const T*)a.t[k].x + b * a.t[k].xs[0] + i * a.t[k].xs[2];
    o[k] = (T*)a.t[k].out + b * a.t[k].os[0] + i * a.t[k].os[2];
  }
  Vec<T, V> va[kRopeFlight], vb[kRopeFlight];
  // item -> its tensor, head and unit; the first of its elements (a pair's
  // other half is `gap` further, nothing behind rot)
  auto place = [&](int item, int& k, int64_t& h, int& u, int& c) {
    k = item >= a.items0;
    const int q = item - (k ? a.items0 : 0);
    h = q / a.units;
    u = q - (int)h * a.units;
    c = u >= a.pair_units ? a.rot + (u - a.pair_units) * V : INTER ? u * 2 * V : u * V;
  };
  const int gap = INTER ? V : a.rot / 2;
  auto load = [&](int base) {
#pragma unroll
    for (int f = 0; f < kRopeFlight; ++f) {
      const int item = base + 32 * f;
      if (item >= a.items) break;
      int k, u, c;
      int64_t h;
      place(item, k, h, u, c);
      const T* src = (k ? x[1] : x[0]) + h * a.t[k].xs[1] + c;
      va[f].load(src);
      if (u < a.pair_units) vb[f].load(src + gap);
    }
  };
  load(lane);
  const double p = (double)a.pos[b * a.pos_stride + i];
  for (int k = lane; k < a.rot / 2; k += 32) {
    // freq / 2 pi and its product with p each as a double and what it rounds off
    const double f = a.freqs[k], g = f * kTurn, g_low = fma(f, kTurn, -g) + f * kTurnLow;
    double turns = p * g;
    const double low = fma(p, g, -turns) + p * g_low;
    turns = (turns - rint(turns)) + low;
    float2 t;
    sincospif(2.f * (float)turns, &t.y, &t.x);
    turn[k] = make_float2(t.x * a.mscale, t.y * (a.inverse ? -a.mscale : a.mscale));
  }
  __syncwarp();
  for (int base = lane; base < a.items; base += 32 * kRopeFlight) {
    if (base != lane) load(base);
#pragma unroll
    for (int f = 0; f < kRopeFlight; ++f) {
      const int item = base + 32 * f;
      if (item >= a.items) break;
      int k, u, c;
      int64_t h;
      place(item, k, h, u, c);
      T* dst = (k ? o[1] : o[0]) + h * a.t[k].os[1] + c;
      if (u < a.pair_units) {
        if constexpr (INTER) {
          float e[2 * V];
#pragma unroll
          for (int q = 0; q < V; ++q) {
            e[q] = to_f32(va[f].e[q]);
            e[V + q] = to_f32(vb[f].e[q]);
          }
#pragma unroll
          for (int q = 0; q < V; ++q) {
            const float2 t = turn[u * V + q];
            const float xa = e[2 * q], xb = e[2 * q + 1];
            e[2 * q] = xa * t.x - xb * t.y;
            e[2 * q + 1] = xb * t.x + xa * t.y;
          }
#pragma unroll
          for (int q = 0; q < V; ++q) {
            va[f].e[q] = from_f32<T>(e[q]);
            vb[f].e[q] = from_f32<T>(e[V + q]);
          }
        } else {
#pragma unroll
          for (int q = 0; q < V; ++q) {
            const float2 t = turn[u * V + q];
            const float xa = to_f32(va[f].e[q]), xb = to_f32(vb[f].e[q]);
            va[f].e[q] = from_f32<T>(xa * t.x - xb * t.y);
            vb[f].e[q] = from_f32<T>(xb * t.x + xa * t.y);
          }
        }
        vb[f].store(dst + gap);
      }
      va[f].store(dst);
    }
  }
}

namespace {

template <typename T, int V>
int rope_launch(RopeArgs& a, int count, bool inter, cudaStream_t s) {
  a.pair_units = a.rot / 2 / V;
  a.units = a.pair_units + (a.d - a.rot) / V;
  const int64_t blocks = (a.rows + kRopeWarps - 1) / kRopeWarps;
  const int64_t items0 = a.t[0].heads * a.units, items1 = count > 1 ? a.t[1].heads * a.units : 0;
  if (blocks > 0x7fffffff || items0 + items1 > 0x3fffffff) return fail(AMC_ERR_INVALID, "amc_rope: too many rows or elements a row");
  a.items0 = (int)items0;
  a.items = (int)(items0 + items1);
  const size_t sm = (size_t)kRopeWarps * (a.rot / 2) * sizeof(float2);
  if (inter) k_rope<T, V, true><<<(unsigned)blocks, kRopeWarps * 32, sm, s>>>(a);
  else k_rope<T, V, false><<<(unsigned)blocks, kRopeWarps * 32, sm, s>>>(a);
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
  if (batch < 0 || n < 0 || d <= 0 || rot <= 0 || rot > d || rot % 2 || rot > kRopeMaxRot)
    return fail(AMC_ERR_INVALID, "amc_rope: bad sizes (rot even, 2..d, at most 1024)");
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
  if (count == 2 && t[0].heads && t[1].heads &&
      (t[0].out == t[1].out || t[0].out == t[1].x || t[1].out == t[0].x))
    return fail(AMC_ERR_INVALID, "amc_rope: the tensors' results must not lie on one another's");
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
