// Shared by the differential-attention translation units.
#pragma once

#include <cmath>

#include "amc_half.cuh"
#include "amc_internal.h"

namespace amc {

// Rows' visible keys are a prefix: row i sees the keys j < diff_limit().
struct DiffLens {
  int nq, nk;   // this sequence's lengths, within the tensors
};

__device__ __forceinline__ DiffLens diff_lens(const amc_diff_attention& p, int b) {
  DiffLens l{p.nq, p.nk};
  if (p.q_lens) l.nq = min(max(p.q_lens[b], 0), p.nq);
  if (p.kv_lens) l.nk = min(max(p.kv_lens[b], 0), p.nk);
  return l;
}
__device__ __forceinline__ int diff_limit(const DiffLens& l, int causal, int i) {
  if (i >= l.nq) return 0;
  return causal ? min(l.nk, max(0, i + l.nk - l.nq + 1)) : l.nk;
}
// The first row that sees key j (nq when none does).
__device__ __forceinline__ int diff_first_row(const DiffLens& l, int causal, int j) {
  if (j >= l.nk) return l.nq;
  return causal ? min(l.nq, max(0, j - (l.nk - l.nq))) : 0;
}

// The natural-log row log-sum-exp from a row's maximum (log2 units) and sum: -inf
// only where nothing was summed, so that a NaN among the scores stays one.
__device__ __forceinline__ float row_lse(float top, float sum) {
  return sum == 0.f ? -INFINITY : fmaf(top, 0.69314718055994530942f, logf(sum));
}

// Workspace of the backward.  For every two rows (2 r, 2 r + 1) of a (batch,
// head) one float4 of each kind, negated for the fused operations that use
// them, both rows of map 1 and then both of map 2:
//   nlse = -lse * log2 e, -inf where the row is empty, so that
//          exp2(s + nlse) is 0
//   nsum = -D_m, D_m = rowsum(dO * O_m)
// (rows padded to a multiple of 4, so that a tile of them is a bulk copy),
// then lam and a counter for every head, then one partial of sum P_2 G for
// every (head, batch, row tile).
//
// fp16 tensors on the tensor cores have the operands that the threads make in
// fp16 too, whose range (2^-24 .. 65504) dS = P (G - D) leaves easily: upstream
// gradients of 2^-17 over 2000 keys came out wrong by twice the rounding of
// their terms.  So dS and P_1 - lam P_2 are formed times powers of two, the same
// for all that add up in a CTA, and the sums are scaled back in f32.  `peaks`
// holds what bounds them: for every (batch, key head) the largest |dO row|^2 and
// |V row|^2, for every key head the largest |lam|, as bits (a maximum's order does
// not change it).
constexpr int kDiffTile = 32;
struct DiffBwdWork {
  float4* nlse;
  float4* nsum;
  float* lam;
  unsigned* done;      // CTAs of this row of lam that have written their partials
  float* partials;
  unsigned* peaks;     // null: nothing is scaled
  int pitch;   // rows of a (batch, head)
};
// The value of row r of map m in such an array.
__device__ __forceinline__ float diff_row(const float4* x, int64_t first_row, int r, int m) {
  return reinterpret_cast<const float*>(x + (first_row + r) / 2)[2 * m + (r & 1)];
}
inline int diff_row_pitch(const amc_diff_attention& p) { return (p.nq + 3) & ~3; }
inline size_t diff_peaks(const amc_diff_attention& p) {
  return p.dtype == AMC_F16 ? (size_t)(2 * p.batch + 1) * p.kv_heads : 0;
}
inline size_t diff_bwd_bytes(const amc_diff_attention& p) {
  const size_t rows = (size_t)p.batch * p.heads * diff_row_pitch(p);
  const size_t partials = (size_t)p.batch * p.heads * ((p.nq + kDiffTile - 1) / kDiffTile);
  return rows * sizeof(float4) + 2 * (size_t)p.heads * sizeof(float) + partials * sizeof(float) +
         diff_peaks(p) * sizeof(unsigned);
}
inline DiffBwdWork diff_bwd_work(const amc_diff_attention& p) {
  const size_t rows = (size_t)p.batch * p.heads * diff_row_pitch(p);
  DiffBwdWork w;
  w.nlse = (float4*)p.workspace;
  w.nsum = w.nlse + rows / 2;
  w.lam = (float*)(w.nsum + rows / 2);
  w.done = (unsigned*)(w.lam + p.heads);
  w.partials = (float*)(w.done + p.heads);
  w.peaks = (unsigned*)(w.partials + (size_t)p.batch * p.heads * ((p.nq + kDiffTile - 1) / kDiffTile));
  w.pitch = diff_row_pitch(p);
  return w;
}
// The exponents of those powers for (batch b, key head g): of dS, which
// |dO| |V| max(1, |lam|) 2 bounds, and of P_1 - lam P_2, bounded by 1 + |lam|; the
// bounds land in 2^14 .. 2^15.  0 where a bound is 0 or not finite.
struct DiffShift {
  int ds, w;
};
__device__ __forceinline__ float diff_pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ DiffShift diff_shift(const amc_diff_attention& p, const DiffBwdWork& w, int b, int g) {
  const unsigned* x = w.peaks + 2 * ((int64_t)b * p.kv_heads + g);
  const float lam = __uint_as_float(w.peaks[2 * (int64_t)p.batch * p.kv_heads + g]);
  auto up = [](float bound) {
    const int e = (int)(__float_as_uint(bound) >> 23) - 127;
    return bound > 0.f && e < 128 ? max(-60, min(60, 14 - e)) : 0;
  };
  return {up(sqrtf(__uint_as_float(x[0])) * sqrtf(__uint_as_float(x[1])) * 2.f * fmaxf(1.f, lam)), up(1.f + lam)};
}

// Tensor-core forward; *handled = false (and nothing launched) for other
// types, shapes and alignments.
bool diff_tc_shape(const amc_diff_attention& p);
int diff_fwd_tc(const amc_diff_attention& p, cudaStream_t s, bool* handled);
// The form for few rows and many keys, likewise, and its workspace.
size_t diff_split_bytes(const amc_diff_attention& p);
int diff_fwd_split(const amc_diff_attention& p, cudaStream_t s, bool* handled);
int launch_diff_fwd_simt(const amc_diff_attention& p, cudaStream_t s);
// CTAs of a cluster that share the query heads of a key head in dK/dV: more
// than one while `ctas`, one for each key tile of a key head, leave SMs idle
// (6 heads over 2 at 5 x 1000 rows take 80).
int diff_share(const amc_diff_attention& p, int64_t ctas);
int launch_diff_bwd_rows(const amc_diff_attention& p, const DiffBwdWork& w, cudaStream_t s);
int launch_diff_bwd_simt(const amc_diff_attention& p, const DiffBwdWork& w, cudaStream_t s);
// Tensor-core gradients (with the rows), likewise.
int diff_bwd_tc(const amc_diff_attention& p, const DiffBwdWork& w, cudaStream_t s, bool* handled);

// exp(l0 . l1) and exp(l2 . l3) of row `row` of lam, on every lane of a converged warp.
template <typename T>
__device__ __forceinline__ float2 lam_exps(const amc_diff_attention& p, int row) {
  const T* l = (const T*)p.lam + (size_t)row * 4 * p.d;
  float a = 0.f, c = 0.f;
  for (int i = threadIdx.x & 31; i < p.d; i += 32) {
    a = fmaf(to_f32(l[i]), to_f32(l[p.d + i]), a);
    c = fmaf(to_f32(l[2 * p.d + i]), to_f32(l[3 * p.d + i]), c);
  }
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  return make_float2(expf(a), expf(c));
}
// lam of head h, likewise.
template <typename T>
__device__ __forceinline__ float lam_of(const amc_diff_attention& p, int h) {
  const float2 e = lam_exps<T>(p, p.lam_rows == 1 ? 0 : h);
  return e.x - e.y + p.lam_init;
}

// A row of dlam from its partials of sum P_2 G, by the first 256 threads of a
// CTA that all call it: a fixed order of summation, in double.
template <typename T>
__device__ __forceinline__ void diff_dlam_row(const amc_diff_attention& p, const DiffBwdWork& w, int row, int tiles,
                                              double* red) {
  const int64_t per_head = (int64_t)p.batch * tiles, n = p.lam_rows == 1 ? per_head * p.heads : per_head;
  const float* x = w.partials + row * per_head;
  double t = 0.0;
  if (threadIdx.x < 256) {
    for (int64_t i = threadIdx.x; i < n; i += 256) t += __ldcg(x + i);
    red[threadIdx.x] = t;
  }
  __syncthreads();
  for (int k = 128; k > 0; k >>= 1) {
    if (threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
    __syncthreads();
  }
  const float dl = (float)-red[0];
  const float2 e = lam_exps<T>(p, row);
  const T* l = (const T*)p.lam + (size_t)row * 4 * p.d;
  T* o = (T*)p.dlam + (size_t)row * 4 * p.d;
  for (int i = threadIdx.x; i < p.d; i += blockDim.x) {
    o[i] = from_f32<T>(dl * e.x * to_f32(l[p.d + i]));
    o[p.d + i] = from_f32<T>(dl * e.x * to_f32(l[i]));
    o[2 * p.d + i] = from_f32<T>(-dl * e.y * to_f32(l[3 * p.d + i]));
    o[3 * p.d + i] = from_f32<T>(-dl * e.y * to_f32(l[2 * p.d + i]));
  }
}
// Called by every dQ CTA of head h after it has written its partial: the last
// of its row of lam (the rows' kernel zeroed the counter) makes that row of
// dlam.  `red`: 256 doubles of shared memory.
template <typename T>
__device__ __forceinline__ void diff_dlam_last(const amc_diff_attention& p, const DiffBwdWork& w, int h, int tiles,
                                               double* red) {
  __shared__ int last;
  const int row = p.lam_rows == 1 ? 0 : h;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned all = (unsigned)((int64_t)p.batch * tiles * (p.lam_rows == 1 ? p.heads : 1));
    last = atomicAdd(w.done + row, 1u) == all - 1;
    __threadfence();
  }
  __syncthreads();
  if (last) diff_dlam_row<T>(p, w, row, tiles, red);
}

}  // namespace amc
