// Differential attention, entry points and the kernels of every case:
//   P_m = softmax(scale Q_m K_m^T), m = 1, 2;  O = (P_1 - lam P_2) V
// with lam = exp(l0.l1) - exp(l2.l3) + lam_init per head.
// Backward, from the rows' log-sum-exps and D_m = rowsum(dO * O_m), G = dO V^T:
//   dS_1 = P_1 (G - D_1)          dS_2 = -lam P_2 (G - D_2)
//   dQ_m = scale dS_m K_m         dK_m = scale dS_m^T Q_m
//   dV   = (P_1 - lam P_2)^T dO   dlam = -sum over rows of D_2
// dlam is summed from P_2 G of the rebuilt map, in f32 before any rounding to
// 16 bits, not from the stored O_2.
//
// These kernels keep everything in f32 on the FMA pipes: a CTA of 16 x 16
// threads owns TT rows (or keys), streams TT-wide tiles of the other side
// through shared memory, and each thread owns a (TT/16)^2 patch of a score
// tile and TT/16 rows x DV/16 columns of an output.  They run f32 tensors,
// where a tensor core would round the operands, and the shapes the
// tensor-core kernels do not take.
//
// Bound: the FMA pipe, 128 a clock and SM, and beside it the reads of shared
// memory: products go by twos (fma.rn.f32x2), which leaves the issue slots to
// them, and the forward's two maps share each read of V (216 -> 187 us for 4 x 8
// heads, 512 x 512, d 64; the FMAs alone take 89 us, 103 with 256 CTAs on 148
// SMs).  16 warps instead of 8, a map each half, gained nothing.  2048 x 2048:
// 2.46 ms, 58 % of the FMA rate.
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "amc_diffattn.h"
#include "amc_half.cuh"
#include "amc_tc.cuh"

namespace amc {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// rows r0 .. r0+TT of a (rows, dim) matrix into dst[TT][W], zero outside
// rows < rows_end and columns < dim.  f32 rows on 16-byte boundaries are
// copied asynchronously (complete at tile_wait), others converted on the way.
template <typename T, int TT, int W, int PITCH>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t stride, int r0, int rows_end, int dim) {
  if constexpr (sizeof(T) == 4) {
    if (!((uintptr_t)src & 15) && stride % 4 == 0 && dim % 4 == 0) {
      for (int i = threadIdx.x; i < TT * W / 4; i += 256) {
        const int r = i / (W / 4), c = i % (W / 4) * 4;
        const bool in = r0 + r < rows_end && c < dim;
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst + r * PITCH + c);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                     ::"r"(to), "l"(in ? src + (int64_t)(r0 + r) * stride + c : src), "r"(in ? 16 : 0) : "memory");
      }
      return;
    }
  }
  for (int i = threadIdx.x; i < TT * W; i += 256) {
    const int r = i / W, c = i % W;
    dst[r * PITCH + c] = (r0 + r < rows_end && c < dim) ? to_f32(src[(int64_t)(r0 + r) * stride + c]) : 0.f;
  }
}
__device__ __forceinline__ void tile_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the latest `N` committed loads of this thread are complete.
template <int N>
__device__ __forceinline__ void tile_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// acc[i][j] += sum_c A[ty + 16 i][c] B[tx + 16 j][c]
template <int R, int PITCH>
__device__ __forceinline__ void dot_rows(float (&acc)[R][R], const float* A, const float* B, int dim, int ty, int tx) {
  float2 acc2[R][R];   // sums of even and of odd columns
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc2[i][j] = make_float2(acc[i][j], 0.f);
  for (int c = 0; c < dim; c += 4) {
    float4 a[R], b[R];
#pragma unroll
    for (int i = 0; i < R; ++i) a[i] = *reinterpret_cast<const float4*>(A + (ty + 16 * i) * PITCH + c);
#pragma unroll
    for (int j = 0; j < R; ++j) b[j] = *reinterpret_cast<const float4*>(B + (tx + 16 * j) * PITCH + c);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < R; ++j)
        acc2[i][j] = tc::fma2(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y),
                              tc::fma2(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w), acc2[i][j]));
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = acc2[i][j].x + acc2[i][j].y;
}

// out[i][4 g + e] += sum_k W(row i, k) X[k][4 tx + 64 g + e].  W is
// w[row * PW + k] with rows ty + 16 i, or transposed w[k * PW + row] with rows
// R ty + i: either way one access brings several of its values.  The R rows are
// those of M matrices W, PM values apart, on the same X.
template <int R, int NC, int TT, int PW, int PX, bool TRANS, int M = 1, int PM = 0>
__device__ __forceinline__ void mul_rows(float (&out)[R][NC], const float* w, const float* X, int ty, int tx) {
  auto step = [&](const float (&a)[R], int k) {
#pragma unroll
    for (int g = 0; g < NC / 4; ++g) {
      const float4 x = *reinterpret_cast<const float4*>(X + k * PX + 4 * tx + 64 * g);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float2 aa = make_float2(a[i], a[i]);
        const float2 lo = tc::fma2(aa, make_float2(x.x, x.y), make_float2(out[i][4 * g], out[i][4 * g + 1]));
        const float2 hi = tc::fma2(aa, make_float2(x.z, x.w), make_float2(out[i][4 * g + 2], out[i][4 * g + 3]));
        out[i][4 * g] = lo.x;
        out[i][4 * g + 1] = lo.y;
        out[i][4 * g + 2] = hi.x;
        out[i][4 * g + 3] = hi.y;
      }
    }
  };
  if constexpr (TRANS) {
#pragma unroll 4
    for (int k = 0; k < TT; ++k) {
      float a[R];
      if constexpr (R == 4) {
        const float4 v = *reinterpret_cast<const float4*>(w + k * PW + 4 * ty);
        a[0] = v.x; a[1] = v.y; a[2] = v.z; a[3] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(w + k * PW + 2 * ty);
        a[0] = v.x; a[1] = v.y;
      }
      step(a, k);
    }
  } else {
#pragma unroll 2
    for (int k = 0; k < TT; k += 4) {
      float4 v[R];
#pragma unroll
      for (int i = 0; i < R; ++i)
        v[i] = *reinterpret_cast<const float4*>(w + i / (R / M) * PM + (ty + 16 * (i % (R / M))) * PW + k);
      float a[R];
#pragma unroll
      for (int i = 0; i < R; ++i) a[i] = v[i].x;
      step(a, k);
#pragma unroll
      for (int i = 0; i < R; ++i) a[i] = v[i].y;
      step(a, k + 1);
#pragma unroll
      for (int i = 0; i < R; ++i) a[i] = v[i].z;
      step(a, k + 2);
#pragma unroll
      for (int i = 0; i < R; ++i) a[i] = v[i].w;
      step(a, k + 3);
    }
  }
}

// Rows as mul_rows has them.
template <typename T, int R, int NC, bool TRANS>
__device__ __forceinline__ void store_rows(T* dst, int64_t stride, const float (*v)[NC], float f, int r0, int rows,
                                           int dim, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + (TRANS ? R * ty + i : ty + 16 * i);
    if (r >= rows) continue;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = 4 * tx + 64 * (c / 4) + (c % 4);
      if (col < dim) dst[(int64_t)r * stride + col] = from_f32<T>(v[i][c] * f);
    }
  }
}

template <int TT, int DM, int DV>
struct Tile {
  static constexpr int R = TT / 16, PD = DM + 4, PV = DV + 4, PP = TT + 4;
  static constexpr int stage = 2 * TT * PD + TT * PV;   // K_1, K_2 and V of the forward's streamed tile
  static constexpr int fwd = (2 * TT * PD + 2 * stage + 2 * TT * PP) * 4;
  static constexpr int dkv = (4 * TT * PD + 2 * TT * PV + 3 * TT * PP) * 4;
  static constexpr int dq = (4 * TT * PD + 2 * TT * PV + 2 * TT * PP) * 4;
};

}  // namespace

template <typename T, int TT, int DM, int DV>
__global__ void __launch_bounds__(256, 1) k_diff_fwd_simt(const __grid_constant__ amc_diff_attention p) {
  using L = Tile<TT, DM, DV>;
  constexpr int R = L::R;
  extern __shared__ float diff_sm[];
  float *sQ = diff_sm, *sP = sQ + 2 * TT * L::PD, *stages = sP + 2 * TT * L::PP;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int r0 = blockIdx.x * TT, h = blockIdx.y, b = blockIdx.z, g = h / (p.heads / p.kv_heads);
  const DiffLens len = diff_lens(p, b);
  const float lam = lam_of<T>(p, h);
  const float c2 = p.scale * kLog2e;
  const int dim4 = (p.d + 3) & ~3;
  for (int m = 0; m < 2; ++m)
    load_tile<T, TT, DM, L::PD>(sQ + m * TT * L::PD, (const T*)p.q + b * p.qs[0] + (2 * h + m) * p.qs[1], p.qs[2], r0,
                                len.nq, p.d);
  int lim[R];
  float top[2][R], sum[2][R], o[2 * R][DV / 16];   // rows of map m from m R on
#pragma unroll
  for (int i = 0; i < R; ++i) {
    lim[i] = diff_limit(len, p.causal, r0 + ty + 16 * i);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      top[m][i] = -INFINITY;
      sum[m][i] = 0.f;
#pragma unroll
      for (int c = 0; c < DV / 16; ++c) o[m * R + i][c] = 0.f;
    }
  }
  const int last = min(r0 + TT, len.nq) - 1;
  const int kend = last >= r0 ? diff_limit(len, p.causal, last) : 0;
  auto load = [&](int k0, int buf) {
    float* st = stages + buf * L::stage;
    for (int m = 0; m < 2; ++m)
      load_tile<T, TT, DM, L::PD>(st + m * TT * L::PD, (const T*)p.k + b * p.ks[0] + (2 * g + m) * p.ks[1], p.ks[2], k0,
                                  len.nk, p.d);
    load_tile<T, TT, DV, L::PV>(st + 2 * TT * L::PD, (const T*)p.v + b * p.vs[0] + g * p.vs[1], p.vs[2], k0, len.nk, p.dv);
  };
  if (kend > 0) load(0, 0);
  tile_commit();
  for (int k0 = 0, buf = 0; k0 < kend; k0 += TT, buf ^= 1) {
    __syncthreads();   // the tile before is used up
    if (k0 + TT < kend) load(k0 + TT, buf ^ 1);
    tile_commit();
    tile_wait<1>();
    __syncthreads();
    const float *sK = stages + buf * L::stage, *sV = sK + 2 * TT * L::PD;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float s[R][R] = {};
      dot_rows<R, L::PD>(s, sQ + m * TT * L::PD, sK + m * TT * L::PD, dim4, ty, tx);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float mx = top[m][i];
#pragma unroll
        for (int j = 0; j < R; ++j) {
          s[i][j] = k0 + tx + 16 * j < lim[i] ? s[i][j] * c2 : -INFINITY;
          mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float base = mx == -INFINITY ? 0.f : mx;   // a row that has seen no key yet
        const float corr = exp2f(top[m][i] - base);
        float add = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const float e = exp2f(s[i][j] - base);
          add += e;
          sP[m * TT * L::PP + (ty + 16 * i) * L::PP + tx + 16 * j] = e;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) add += __shfl_xor_sync(0xffffffffu, add, w);
        sum[m][i] = sum[m][i] * corr + add;
        top[m][i] = mx;
#pragma unroll
        for (int c = 0; c < DV / 16; ++c) o[m * R + i][c] *= corr;
      }
    }
    __syncthreads();
    mul_rows<2 * R, DV / 16, TT, L::PP, L::PV, false, 2, TT * L::PP>(o, sP, sV, ty, tx);
  }
  tile_wait<0>();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + ty + 16 * i;
    float inv[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      inv[m] = sum[m][i] != 0.f ? 1.f / sum[m][i] : 0.f;
      if (p.lse && tx == 0 && r < p.nq)
        p.lse[((int64_t)b * 2 * p.heads + 2 * h + m) * p.nq + r] =
            row_lse(top[m][i], sum[m][i]);
    }
#pragma unroll
    for (int c = 0; c < DV / 16; ++c) {
      o[R + i][c] *= inv[1];
      o[i][c] = fmaf(-lam, o[R + i][c], o[i][c] * inv[0]);
    }
  }
  store_rows<T, R, DV / 16, false>((T*)p.o + b * p.os[0] + h * p.os[1], p.os[2], o, 1.f, r0, p.nq, p.dv, ty, tx);
  if (p.o2) store_rows<T, R, DV / 16, false>((T*)p.o2 + b * p.o2s[0] + h * p.o2s[1], p.o2s[2], o + R, 1.f, r0, p.nq, p.dv, ty, tx);
}

// nlse and nsum from lse, o, o2 and dO, and lam of every head.  A row is
// shared by LANES lanes of V elements a load (16 bytes where every row is
// aligned): the pass reads three output-sized tensors once and is bound by
// that.
template <typename T, int V, int LANES>
__global__ void __launch_bounds__(256) k_diff_bwd_rows(const __grid_constant__ amc_diff_attention p,
                                                       const __grid_constant__ DiffBwdWork w) {
  constexpr int kAtOnce = 2, kRows = 256 / LANES;   // rows in flight a thread, rows of a CTA at a time
  const int sub = threadIdx.x % LANES, h = blockIdx.y, b = blockIdx.z;
  const int i0 = blockIdx.x * kAtOnce * kRows + threadIdx.x / LANES;
  const DiffLens len = diff_lens(p, b);
  float up = 0.f;   // P is rebuilt times 2^up
  if constexpr (std::is_same<T, __half>::value)
    if (w.peaks) up = (float)diff_shift(p, w, b, h / (p.heads / p.kv_heads)).ds;
  float d[kAtOnce] = {}, d2[kAtOnce] = {}, nl1[kAtOnce], nl2[kAtOnce];
#pragma unroll
  for (int r = 0; r < kAtOnce; ++r) {
    const int i = i0 + r * kRows;
    nl1[r] = nl2[r] = -INFINITY;
    if (i < p.nq && diff_limit(len, p.causal, i) > 0) {
      const float* lse = p.lse + ((int64_t)b * 2 * p.heads + 2 * h) * p.nq + i;
      // a row whose scores are all -inf has -inf here too: like a row that sees no key
      nl1[r] = lse[0] == -INFINITY ? -INFINITY : fmaf(-lse[0], kLog2e, up);
      nl2[r] = lse[p.nq] == -INFINITY ? -INFINITY : fmaf(-lse[p.nq], kLog2e, up);
      const T* o = (const T*)p.o + b * p.os[0] + h * p.os[1] + (int64_t)i * p.os[2];
      const T* o2 = (const T*)p.o2 + b * p.o2s[0] + h * p.o2s[1] + (int64_t)i * p.o2s[2];
      const T* go = (const T*)p.d_o + b * p.dos[0] + h * p.dos[1] + (int64_t)i * p.dos[2];
      for (int c = sub * V; c < p.dv; c += LANES * V) {
        if constexpr (V == 8) {
          const uint4 x = *reinterpret_cast<const uint4*>(go + c), y = *reinterpret_cast<const uint4*>(o + c),
                      z = *reinterpret_cast<const uint4*>(o2 + c);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 a = unpack2<T>(xs[k]), e = unpack2<T>(ys[k]), f = unpack2<T>(zs[k]);
            d[r] = fmaf(a.x, e.x, fmaf(a.y, e.y, d[r]));
            d2[r] = fmaf(a.x, f.x, fmaf(a.y, f.y, d2[r]));
          }
        } else {
          const float x = to_f32(go[c]);
          d[r] = fmaf(x, to_f32(o[c]), d[r]);
          d2[r] = fmaf(x, to_f32(o2[c]), d2[r]);
        }
      }
    }
  }
  const float lam = lam_of<T>(p, h);   // after the loads, not before them
  if (blockIdx.x == 0 && b == 0 && threadIdx.x == 0) {
    w.lam[h] = lam;
    w.done[h] = 0;
  }
#pragma unroll
  for (int r = 0; r < kAtOnce; ++r) {
#pragma unroll
    for (int s = LANES / 2; s > 0; s >>= 1) {
      d[r] += __shfl_xor_sync(0xffffffffu, d[r], s);
      d2[r] += __shfl_xor_sync(0xffffffffu, d2[r], s);
    }
    const int i = i0 + r * kRows;
    if (sub == 0 && i < w.pitch) {   // the padding too: the gradients multiply it by 0
      const int64_t at = ((int64_t)b * p.heads + h) * w.pitch + i;
      float* e = reinterpret_cast<float*>(w.nlse + at / 2) + (at & 1);
      float* n = reinterpret_cast<float*>(w.nsum + at / 2) + (at & 1);
      e[0] = nl1[r];
      e[2] = nl2[r];
      n[0] = -fmaf(lam, d2[r], d[r]);   // dO . O_1 = dO . (O + lam O_2)
      n[2] = -d2[r];
    }
  }
}

// dK, dV of TT keys of one key head: streams the rows of its query heads.  Its
// heads are shared by the `share` CTAs of a cluster, which add their parts up
// in order of rank (as in the tensor-core kernel).
template <typename T, int TT, int DM, int DV>
__global__ void __launch_bounds__(256, 1) k_diff_dkv_simt(const __grid_constant__ amc_diff_attention p,
                                                          const __grid_constant__ DiffBwdWork wk, int share) {
  using L = Tile<TT, DM, DV>;
  constexpr int R = L::R;
  extern __shared__ float diff_sm[];
  float *sK = diff_sm, *sQ = sK + 2 * TT * L::PD, *sV = sQ + 2 * TT * L::PD, *sG = sV + TT * L::PV;
  float *sB = sG + TT * L::PV, *sS = sB + TT * L::PP;   // P_1 - lam P_2, then dS_1 and dS_2, as [row][key]
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int k0 = blockIdx.x / share * TT, rank = blockIdx.x % share, g = blockIdx.y, b = blockIdx.z;
  const int heads = p.heads / p.kv_heads / share, head0 = (g * share + rank) * heads;
  const DiffLens len = diff_lens(p, b);
  const float c2 = p.scale * kLog2e;
  const int dim4 = (p.d + 3) & ~3, dimv4 = (p.dv + 3) & ~3;
  for (int m = 0; m < 2; ++m)
    load_tile<T, TT, DM, L::PD>(sK + m * TT * L::PD, (const T*)p.k + b * p.ks[0] + (2 * g + m) * p.ks[1], p.ks[2], k0,
                                len.nk, p.d);
  load_tile<T, TT, DV, L::PV>(sV, (const T*)p.v + b * p.vs[0] + g * p.vs[1], p.vs[2], k0, len.nk, p.dv);
  float dk[2][R][DM / 16] = {}, dv[R][DV / 16] = {};
  const int first = diff_first_row(len, p.causal, k0) / TT * TT;
  for (int h = head0; h < head0 + heads; ++h) {
    const float lam = wk.lam[h];
    for (int r0 = first; r0 < len.nq; r0 += TT) {
      __syncthreads();
      for (int m = 0; m < 2; ++m)
        load_tile<T, TT, DM, L::PD>(sQ + m * TT * L::PD, (const T*)p.q + b * p.qs[0] + (2 * h + m) * p.qs[1], p.qs[2],
                                    r0, len.nq, p.d);
      load_tile<T, TT, DV, L::PV>(sG, (const T*)p.d_o + b * p.dos[0] + h * p.dos[1], p.dos[2], r0, len.nq, p.dv);
      tile_commit();
      tile_wait<0>();
      __syncthreads();
      float gv[R][R] = {}, both[R][R];
      dot_rows<R, L::PV>(gv, sG, sV, dimv4, ty, tx);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float s[R][R] = {};
        dot_rows<R, L::PD>(s, sQ + m * TT * L::PD, sK + m * TT * L::PD, dim4, ty, tx);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int r = r0 + ty + 16 * i;
          const int lim = diff_limit(len, p.causal, r);
          const int64_t at = ((int64_t)b * p.heads + h) * wk.pitch;
          const float e = lim > 0 ? diff_row(wk.nlse, at, r, m) : -INFINITY;
          const float ds = lim > 0 ? diff_row(wk.nsum, at, r, m) : 0.f;
#pragma unroll
          for (int j = 0; j < R; ++j) {
            const float pr = k0 + tx + 16 * j < lim ? exp2f(fmaf(s[i][j], c2, e)) : 0.f;
            const float w = m ? -lam * pr : pr;
            both[i][j] = m ? both[i][j] + w : w;
            sS[m * TT * L::PP + (ty + 16 * i) * L::PP + tx + 16 * j] = w * (gv[i][j] + ds);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) sB[(ty + 16 * i) * L::PP + tx + 16 * j] = both[i][j];
      __syncthreads();
      mul_rows<R, DV / 16, TT, L::PP, L::PV, true>(dv, sB, sG, ty, tx);
#pragma unroll
      for (int m = 0; m < 2; ++m)
        mul_rows<R, DM / 16, TT, L::PP, L::PD, true>(dk[m], sS + m * TT * L::PP, sQ + m * TT * L::PD, ty, tx);
    }
  }
  tile_wait<0>();
  if (share > 1) {
    // [map 1 | map 2 | dV] of this CTA, then each CTA's rows of the sum
    constexpr int W = 2 * DM + DV;
    float* part = diff_sm;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float* row = part + (R * ty + i) * W;
#pragma unroll
      for (int c = 0; c < DM / 16; c += 4)
#pragma unroll
        for (int m = 0; m < 2; ++m)
          *reinterpret_cast<float4*>(row + m * DM + 4 * tx + 16 * c) =
              make_float4(dk[m][i][c], dk[m][i][c + 1], dk[m][i][c + 2], dk[m][i][c + 3]);
#pragma unroll
      for (int c = 0; c < DV / 16; c += 4)
        *reinterpret_cast<float4*>(row + 2 * DM + 4 * tx + 16 * c) = make_float4(dv[i][c], dv[i][c + 1], dv[i][c + 2], dv[i][c + 3]);
    }
    tc::cluster_sync();
    const int rows = (TT + share - 1) / share;
    for (int q = threadIdx.x; q < rows * (W / 4); q += 256) {
      const int row = rank * rows + q / (W / 4), c = q % (W / 4) * 4, key = k0 + row;
      if (row >= TT || key >= p.nk) continue;
      float4 sum = tc::ld_cluster(part + row * W + c, 0);
      for (int r = 1; r < share; ++r) {
        const float4 v = tc::ld_cluster(part + row * W + c, r);
        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
      }
      const int m = c / DM, cc = m < 2 ? c % DM : c - 2 * DM, dim = m < 2 ? p.d : p.dv;
      const float f = m < 2 ? p.scale : 1.f;
      T* dst = m < 2 ? (T*)p.dk + b * p.dks[0] + (2 * g + m) * p.dks[1] + (int64_t)key * p.dks[2]
                     : (T*)p.dv_ + b * p.dvs[0] + g * p.dvs[1] + (int64_t)key * p.dvs[2];
      const float s4[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (cc + e < dim) dst[cc + e] = from_f32<T>(s4[e] * f);
    }
    tc::cluster_sync();   // the others have read this CTA's part
    return;
  }
  for (int m = 0; m < 2; ++m)
    store_rows<T, R, DM / 16, true>((T*)p.dk + b * p.dks[0] + (2 * g + m) * p.dks[1], p.dks[2], dk[m], p.scale, k0, p.nk, p.d,
                              ty, tx);
  store_rows<T, R, DV / 16, true>((T*)p.dv_ + b * p.dvs[0] + g * p.dvs[1], p.dvs[2], dv, 1.f, k0, p.nk, p.dv, ty, tx);
}

// dQ of TT rows, and this tile's part of sum P_2 G.
template <typename T, int TT, int DM, int DV>
__global__ void __launch_bounds__(256, 1) k_diff_dq_simt(const __grid_constant__ amc_diff_attention p,
                                                         const __grid_constant__ DiffBwdWork wk) {
  using L = Tile<TT, DM, DV>;
  constexpr int R = L::R;
  extern __shared__ float diff_sm[];
  float *sQ = diff_sm, *sK = sQ + 2 * TT * L::PD, *sG = sK + 2 * TT * L::PD, *sV = sG + TT * L::PV;
  float* sS = sV + TT * L::PV;
  __shared__ float red[8];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int r0 = blockIdx.x * TT, h = blockIdx.y, b = blockIdx.z, g = h / (p.heads / p.kv_heads);
  const DiffLens len = diff_lens(p, b);
  const float lam = wk.lam[h];
  const float c2 = p.scale * kLog2e;
  const int dim4 = (p.d + 3) & ~3, dimv4 = (p.dv + 3) & ~3;
  for (int m = 0; m < 2; ++m)
    load_tile<T, TT, DM, L::PD>(sQ + m * TT * L::PD, (const T*)p.q + b * p.qs[0] + (2 * h + m) * p.qs[1], p.qs[2], r0,
                                len.nq, p.d);
  load_tile<T, TT, DV, L::PV>(sG, (const T*)p.d_o + b * p.dos[0] + h * p.dos[1], p.dos[2], r0, len.nq, p.dv);
  int lim[R];
  float2 e[R], ds[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + ty + 16 * i;
    lim[i] = diff_limit(len, p.causal, r);
    const int64_t at = ((int64_t)b * p.heads + h) * wk.pitch;
    e[i] = make_float2(-INFINITY, -INFINITY);
    ds[i] = make_float2(0.f, 0.f);
    if (lim[i] > 0) {
      e[i] = make_float2(diff_row(wk.nlse, at, r, 0), diff_row(wk.nlse, at, r, 1));
      ds[i] = make_float2(diff_row(wk.nsum, at, r, 0), diff_row(wk.nsum, at, r, 1));
    }
  }
  float dq[2][R][DM / 16] = {}, pg = 0.f;
  const int last = min(r0 + TT, len.nq) - 1;
  const int kend = last >= r0 ? diff_limit(len, p.causal, last) : 0;
  for (int k0 = 0; k0 < kend; k0 += TT) {
    __syncthreads();
    for (int m = 0; m < 2; ++m)
      load_tile<T, TT, DM, L::PD>(sK + m * TT * L::PD, (const T*)p.k + b * p.ks[0] + (2 * g + m) * p.ks[1], p.ks[2], k0,
                                  len.nk, p.d);
    load_tile<T, TT, DV, L::PV>(sV, (const T*)p.v + b * p.vs[0] + g * p.vs[1], p.vs[2], k0, len.nk, p.dv);
    tile_commit();
    tile_wait<0>();
    __syncthreads();
    float gv[R][R] = {}, part = 0.f;
    dot_rows<R, L::PV>(gv, sG, sV, dimv4, ty, tx);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float s[R][R] = {};
      dot_rows<R, L::PD>(s, sQ + m * TT * L::PD, sK + m * TT * L::PD, dim4, ty, tx);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const float pr = k0 + tx + 16 * j < lim[i] ? exp2f(fmaf(s[i][j], c2, m ? e[i].y : e[i].x)) : 0.f;
          if (m) part = fmaf(pr, gv[i][j], part);
          sS[m * TT * L::PP + (ty + 16 * i) * L::PP + tx + 16 * j] =
              (m ? -lam * pr : pr) * (gv[i][j] + (m ? ds[i].y : ds[i].x));
        }
    }
    pg += part;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m)
      mul_rows<R, DM / 16, TT, L::PP, L::PD, false>(dq[m], sS + m * TT * L::PP, sK + m * TT * L::PD, ty, tx);
  }
  tile_wait<0>();
  for (int m = 0; m < 2; ++m)
    store_rows<T, R, DM / 16, false>((T*)p.dq + b * p.dqs[0] + (2 * h + m) * p.dqs[1], p.dqs[2], dq[m], p.scale, r0, p.nq, p.d,
                              ty, tx);
  for (int w = 16; w > 0; w >>= 1) pg += __shfl_xor_sync(0xffffffffu, pg, w);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = pg;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int w = 0; w < 8; ++w) t += red[w];
    wk.partials[((int64_t)h * p.batch + b) * gridDim.x + blockIdx.x] = t;
  }
  diff_dlam_last<T>(p, wk, h, gridDim.x, reinterpret_cast<double*>(diff_sm));
}

// dlam where there are no rows: zeros.
template <typename T>
__global__ void __launch_bounds__(256) k_diff_no_dlam(const __grid_constant__ amc_diff_attention p) {
  for (int64_t i = threadIdx.x; i < (int64_t)p.lam_rows * 4 * p.d; i += 256) ((T*)p.dlam)[i] = from_f32<T>(0.f);
}

int diff_share(const amc_diff_attention& p, int64_t ctas) {
  const int group = p.heads / p.kv_heads;
  int share = 1;
  for (int c = 2; c <= 8 && c <= group && ctas * share < num_sms(); ++c)
    if (group % c == 0) share = c;
  return share;
}

namespace {

template <typename F>
int by_type(int32_t dtype, F f) {
  if (dtype == AMC_F32) return f(float());
  if (dtype == AMC_BF16) return f(__nv_bfloat16());
  return f(__half());
}

template <typename T, int TT, int DM, int DV>
int fwd_simt(const amc_diff_attention& p, cudaStream_t s) {
  static std::atomic<uint64_t> attr{0};
  if (int rc = smem_attr_once(k_diff_fwd_simt<T, TT, DM, DV>, Tile<TT, DM, DV>::fwd, attr)) return rc;
  k_diff_fwd_simt<T, TT, DM, DV><<<dim3((p.nq + TT - 1) / TT, p.heads, p.batch), 256, Tile<TT, DM, DV>::fwd, s>>>(p);
  AMC_CUDA(cudaGetLastError());
  return AMC_OK;
}

template <typename T, int TT, int DM, int DV>
int bwd_simt(const amc_diff_attention& p, const DiffBwdWork& w, cudaStream_t s) {
  static std::atomic<uint64_t> attr_dkv{0}, attr_dq{0};
  using L = Tile<TT, DM, DV>;
  if (int rc = smem_attr_once(k_diff_dkv_simt<T, TT, DM, DV>, L::dkv, attr_dkv)) return rc;
  if (int rc = smem_attr_once(k_diff_dq_simt<T, TT, DM, DV>, L::dq, attr_dq)) return rc;
  if (p.nk) {
    const int key_tiles = (p.nk + TT - 1) / TT;
    const int share = diff_share(p, (int64_t)key_tiles * p.kv_heads * p.batch);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(key_tiles * share, p.kv_heads, p.batch);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = L::dkv;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)share, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = share > 1 ? 1 : 0;
    AMC_CUDA(cudaLaunchKernelEx(&cfg, k_diff_dkv_simt<T, TT, DM, DV>, p, w, share));
  }
  if (p.nq) {
    const int tiles = (p.nq + TT - 1) / TT;
    k_diff_dq_simt<T, TT, DM, DV><<<dim3(tiles, p.heads, p.batch), 256, L::dq, s>>>(p, w);
    AMC_CUDA(cudaGetLastError());
  }
  return AMC_OK;
}

}  // namespace

int launch_diff_fwd_simt(const amc_diff_attention& p, cudaStream_t s) {
  return by_type(p.dtype, [&](auto t) {
    using T = decltype(t);
    return p.d <= 64 && p.dv <= 128 ? fwd_simt<T, 64, 64, 128>(p, s) : fwd_simt<T, 32, 128, 256>(p, s);
  });
}

int launch_diff_bwd_rows(const amc_diff_attention& p, const DiffBwdWork& w, cudaStream_t s) {
  if (!p.nq) return AMC_OK;
  bool wide = p.dtype != AMC_F32 && p.dv % 8 == 0 && !(((uintptr_t)p.o | (uintptr_t)p.o2 | (uintptr_t)p.d_o) & 15);
  const int64_t extent[3] = {p.batch, p.heads, p.nq};
  for (int j = 0; j < 3; ++j) wide = wide && (extent[j] == 1 || (p.os[j] % 8 == 0 && p.o2s[j] % 8 == 0 && p.dos[j] % 8 == 0));
  const dim3 grid16((w.pitch + 31) / 32, p.heads, p.batch), grid8((w.pitch + 15) / 16, p.heads, p.batch);
  if (wide && p.dtype == AMC_BF16) k_diff_bwd_rows<__nv_bfloat16, 8, 16><<<grid16, 256, 0, s>>>(p, w);
  else if (wide) k_diff_bwd_rows<__half, 8, 16><<<grid16, 256, 0, s>>>(p, w);
  else if (p.dtype == AMC_F32) k_diff_bwd_rows<float, 1, 32><<<grid8, 256, 0, s>>>(p, w);
  else if (p.dtype == AMC_BF16) k_diff_bwd_rows<__nv_bfloat16, 1, 32><<<grid8, 256, 0, s>>>(p, w);
  else k_diff_bwd_rows<__half, 1, 32><<<grid8, 256, 0, s>>>(p, w);
  AMC_CUDA(cudaGetLastError());
  return AMC_OK;
}

int launch_diff_bwd_simt(const amc_diff_attention& p, const DiffBwdWork& work, cudaStream_t s) {
  DiffBwdWork w = work;
  w.peaks = nullptr;   // all in f32
  if (int rc = launch_diff_bwd_rows(p, w, s)) return rc;
  return by_type(p.dtype, [&](auto t) {
    using T = decltype(t);
    return p.d <= 64 && p.dv <= 128 ? bwd_simt<T, 64, 64, 128>(p, w, s) : bwd_simt<T, 32, 128, 256>(p, w, s);
  });
}

static int launch_no_dlam(const amc_diff_attention& p, cudaStream_t s) {
  return by_type(p.dtype, [&](auto t) {
    k_diff_no_dlam<decltype(t)><<<1, 256, 0, s>>>(p);
    AMC_CUDA(cudaGetLastError());
    return AMC_OK;
  });
}

namespace {

int check_sizes(const amc_diff_attention* p, const char* who) {
  if (!p) return fail(AMC_ERR_INVALID, std::string(who) + ": null argument");
  if (p->dtype != AMC_F32 && p->dtype != AMC_BF16 && p->dtype != AMC_F16)
    return fail(AMC_ERR_INVALID, std::string(who) + ": dtype must be f32, bf16 or f16");
  if (p->batch < 0 || p->nq < 0 || p->nk < 0 || p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads)
    return fail(AMC_ERR_INVALID, std::string(who) + ": bad sizes (heads must be a multiple of kv_heads)");
  if (p->d <= 0 || p->d > 128 || p->dv <= 0 || p->dv > 256)
    return fail(AMC_ERR_INVALID, std::string(who) + ": head dims d 1..128, dv 1..256");
  if (p->batch > 65535 || p->heads > 32767 || p->nq > (1 << 30) || p->nk > (1 << 30))
    return fail(AMC_ERR_INVALID, std::string(who) + ": batch up to 65535, heads up to 32767, rows up to 2^30");
  if (!std::isfinite(p->scale) || !std::isfinite(p->lam_init))
    return fail(AMC_ERR_INVALID, std::string(who) + ": scale and lam_init must be finite");
  if (p->lam_rows != 1 && p->lam_rows != p->heads)
    return fail(AMC_ERR_INVALID, std::string(who) + ": lam has 1 row or one for each head");
  return AMC_OK;
}

// No result may be another result or something that is read.
int check_results(std::initializer_list<const void*> written, std::initializer_list<const void*> read, const char* who) {
  for (auto w = written.begin(); w != written.end(); ++w) {
    bool twice = false;
    for (auto o = written.begin(); o != w; ++o) twice = twice || (*w && *w == *o);
    for (const void* r : read) twice = twice || (*w && *w == r);
    if (twice) return fail(AMC_ERR_INVALID, std::string(who) + ": a result lies on another tensor of the call");
  }
  return AMC_OK;
}

int check_workspace(const amc_diff_attention* p, size_t need, const char* who) {
  if (!need) return AMC_OK;
  if (!p->workspace || p->workspace_bytes < 0 || (size_t)p->workspace_bytes < need || ((uintptr_t)p->workspace & 15))
    return fail(AMC_ERR_INVALID, std::string(who) + ": workspace of " + std::to_string(need) +
                                     " bytes, 16-byte aligned, expected");
  return AMC_OK;
}

}  // namespace

}  // namespace amc

using namespace amc;

extern "C" {

int amc_diff_attention_workspace(const amc_diff_attention* p, int32_t backward, int64_t* bytes) {
  if (!bytes) return fail(AMC_ERR_INVALID, "amc_diff_attention_workspace: null out");
  if (int rc = check_sizes(p, "amc_diff_attention_workspace")) return rc;
  size_t n = diff_split_bytes(*p);
  if (backward && diff_bwd_bytes(*p) > n) n = diff_bwd_bytes(*p);
  *bytes = (int64_t)n;
  return AMC_OK;
}

int amc_diff_attention_fwd(const amc_diff_attention* p, void* stream) {
  if (int rc = check_sizes(p, "amc_diff_attention_fwd")) return rc;
  if (!p->batch || !p->nq) return AMC_OK;
  if (!p->q || !p->o || !p->lam || (p->nk && (!p->k || !p->v)))
    return fail(AMC_ERR_INVALID, "amc_diff_attention_fwd: null tensor");
  if (int rc = check_workspace(p, diff_split_bytes(*p), "amc_diff_attention_fwd")) return rc;
  if (fault_injected("launch")) return fail(AMC_ERR_INJECTED, "diff_attention: injected launch failure (AMC_FAULT=launch)");
  if (int rc = check_results({p->o, p->o2, p->lse}, {p->q, p->nk ? p->k : nullptr, p->nk ? p->v : nullptr, p->lam},
                             "amc_diff_attention_fwd"))
    return rc;
  cudaStream_t s = pick_stream(stream);
  bool handled = false;
  if (int rc = diff_fwd_split(*p, s, &handled)) return rc;
  if (handled) return AMC_OK;
  if (int rc = diff_fwd_tc(*p, s, &handled)) return rc;
  if (handled) return AMC_OK;
  return launch_diff_fwd_simt(*p, s);
}

int amc_diff_attention_bwd(const amc_diff_attention* p, void* stream) {
  if (int rc = check_sizes(p, "amc_diff_attention_bwd")) return rc;
  if (!p->lam || !p->dlam) return fail(AMC_ERR_INVALID, "amc_diff_attention_bwd: null tensor");
  if (p->batch && ((p->nq && (!p->q || !p->o || !p->o2 || !p->lse || !p->d_o || !p->dq)) ||
                   (p->nk && (!p->k || !p->v || !p->dk || !p->dv_))))
    return fail(AMC_ERR_INVALID, "amc_diff_attention_bwd: null tensor");
  if (int rc = check_workspace(p, diff_bwd_bytes(*p), "amc_diff_attention_bwd")) return rc;
  if (fault_injected("launch")) return fail(AMC_ERR_INJECTED, "diff_attention: injected launch failure (AMC_FAULT=launch)");
  if (p->batch && p->nq && p->nk)
    if (int rc = check_results({p->dq, p->dk, p->dv_, p->dlam},
                               {p->q, p->k, p->v, p->lam, p->o, p->o2, p->lse, p->d_o}, "amc_diff_attention_bwd"))
      return rc;
  cudaStream_t s = pick_stream(stream);
  const DiffBwdWork w = diff_bwd_work(*p);
  if (!p->batch || !p->nq)
    if (int rc = launch_no_dlam(*p, s)) return rc;
  if (!p->batch) return AMC_OK;
  bool handled = false;
  if (int rc = diff_bwd_tc(*p, w, s, &handled)) return rc;
  if (handled) return AMC_OK;
  return launch_diff_bwd_simt(*p, w, s);
}

}  // extern "C"
