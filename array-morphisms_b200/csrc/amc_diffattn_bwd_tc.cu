// Differential attention gradients on the tensor cores (sm_100a, tcgen05
// kind::f16), 16-bit tensors with d <= 64 and dv <= 128, both multiples of 8:
//   P_m = 2^(scale log2e Q_m K_m^T + nlse_m)      G = dO V^T
//   dS_1 = P_1 (G - D_1)                          dS_2 = lam P_2 (D_2 - G)
//   dV = (P_1 - lam P_2)^T dO   dK_m = scale dS_m^T Q_m   dQ_m = scale dS_m K_m
// Both maps share G, and the difference of the maps is taken before dV's
// product, so a (row, key) pair costs 16 d + 12 d operations in two kernels
// against 20 d were dQ added up across CTAs; without atomics the results are
// the same at every call.  One launch holds both kinds of CTA, those of dK/dV
// first, so that neither waits for the other's last ones:
//   dkv_cta        one CTA per 128 keys of a key head; streams 64-row tiles of
//                  every query head that shares it, or, where such CTAs would
//                  not fill the GPU, one cluster of CTAs that take a share of
//                  those heads each and add up through distributed shared
//                  memory, in order of rank;
//   dq_cta         one CTA per 128 rows of a query head; streams 64-key tiles,
//                  and sums P_2 G (dlam) in f32 on the way; the last CTA of a
//                  row of lam adds its partial sums up, in their order.
// The operands that the threads make (the difference of the maps, dS_1, dS_2)
// are rounded to the tensors' type (half a step each, which makes the gradients
// 1.5 times as far from 64 bits as f32 products rounded once; fp16 ones times
// powers of two, see amc_diffattn.h) and stay in tensor memory, written over
// the scores they came from; a thread writes only columns it has read.  A
// 16-bit tile in the 128-byte swizzle serves K-major (its rows as N) and
// MN-major (its rows as K) alike, so one copy of Q, K and dO feeds both
// products.  Four warpgroups share a tile, 16 of its 64 columns each: with two
// of them, 32 columns a thread, the two warps of a scheduler could not cover
// each other's latencies.
// Measured, 8 heads x 16 sequences, 2048 x 2048, d 64, no mask: 1150 us after a
// row pass of 50 us (687 GFLOP counted as 20 d a pair: 600 TFLOP/s).  dkv_cta
// takes 2300 clocks for a 128 x 64 tile, dq_cta 1600; at the rates of either
// alone its products need 1370 and 1110 of them, its exponentials 1024.  The
// rest are the chain from scores through exponentials and G to the operands and
// the round trips at its barriers (200 to 300 clocks each beside the operands of
// the products).  Testing two barriers in one trip, reading the row pairs a tile
// ahead, one wait for both scores, and G of dq_cta behind a barrier of its own
// gained nothing.
// Every wait is bounded; on expiry the kernel records AMC_ERR_TIMEOUT, drains
// and returns.
#include <cmath>
#include <type_traits>

#include "amc_diffattn.h"
#include "amc_half.cuh"
#include "amc_tc.cuh"

namespace amc {

using namespace tc;

namespace {

constexpr int kThreadsB = 576;       // warps 0-15 rows (four warpgroups), 16 loads, 17 issues
constexpr int kRowThreads = 512, kRowWarps = 16;
constexpr int kStages = 4;
constexpr float kLog2e = 1.4426950408889634f;

// dK/dV kernel (bytes from a 1024-aligned base)
template <int NV>
struct KvSmem {
  static constexpr int k = 0;                                 // 2 maps x 128 keys
  static constexpr int v = 32768;
  static constexpr int f = v + NV / 64 * 16384;               // stages: Q_1, Q_2 (8 KB each), dO, pairs
  static constexpr int stage = 16384 + NV / 64 * 8192;
  static constexpr int r = f + kStages * stage;               // stages: 32 nlse, 32 nsum (two rows each)
  static constexpr int bar = r + kStages * 1024;
  static constexpr int bytes = bar + 256 + 1024;
};
// dQ kernel
template <int NV>
struct QSmem {
  static constexpr int q = 0;
  static constexpr int g = 32768;                             // dO
  static constexpr int f = g + NV / 64 * 16384;               // stages: K_1, K_2 (8 KB each), V
  static constexpr int stage = 16384 + NV / 64 * 8192;
  static constexpr int bar = f + kStages * stage;
  static constexpr int bytes = bar + 320 + 1024;
};
constexpr int kPartPitch = 260;      // floats: dK_1, dK_2, dV, and a shift of banks from row to row
static_assert(128 * kPartPitch * 4 <= KvSmem<64>::r, "a cluster's parts fit the tiles' memory");
static_assert(KvSmem<128>::bytes <= 232448 && QSmem<128>::bytes <= 232448, "shared memory");

__device__ int g_diff_bwd_error;

template <typename T>
__device__ __forceinline__ void store16(T* dst, const float (&v)[16], float f, int cols) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack2<T>(v[2 * i] * f, v[2 * i + 1] * f);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (8 * i < cols)
      *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

// Zero the 128-byte row of a swizzled tile region.
__device__ __forceinline__ void zero_row(unsigned char* row) {
#pragma unroll
  for (int i = 0; i < 8; ++i) *reinterpret_cast<int4*>(row + 16 * i) = make_int4(0, 0, 0, 0);
}

}  // namespace

// ------------------------------------------------------------------ what bounds fp16 operands
// The peaks of the workspace, zero before: rows of dO of every head, then rows of
// V of every key head, 64 a CTA, 16 lanes a row.  What is behind the lengths is
// left out, and a NaN, whose row is NaN at any scale.
constexpr int kPeakRows = 64;
__global__ void __launch_bounds__(256) k_diff_peaks(const __grid_constant__ amc_diff_attention p,
                                                    const __grid_constant__ DiffBwdWork w) {
  __shared__ float top[8];
  const bool values = (int)blockIdx.y >= p.heads;
  const int h = values ? blockIdx.y - p.heads : blockIdx.y, b = blockIdx.z;
  const int g = values ? h : h / (p.heads / p.kv_heads), sub = threadIdx.x & 15;
  const DiffLens len = diff_lens(p, b);
  const int64_t* st = values ? p.vs : p.dos;
  const __half* x = (const __half*)(values ? p.v : p.d_o) + b * st[0] + h * st[1];
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < kPeakRows / 16; ++k) {
    const int64_t r = (int64_t)blockIdx.x * kPeakRows + 16 * k + threadIdx.x / 16;
    float n = 0.f;
    if (8 * sub < p.dv && (values ? r < len.nk : r < p.nq && diff_limit(len, p.causal, (int)r) > 0)) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + r * st[2] + 8 * sub);
      const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<__half>(e[i]);
        n = fmaf(f.x, f.x, fmaf(f.y, f.y, n));
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    most = fmaxf(most, n);
  }
  most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) most = fmaxf(most, top[i]);
    atomicMax(w.peaks + 2 * ((int64_t)b * p.kv_heads + g) + values, __float_as_uint(most));
  }
  if (!values && blockIdx.x == 0 && b == 0 && threadIdx.x < 32) {
    const float lam = fabsf(lam_of<__half>(p, h));
    if (threadIdx.x == 0) atomicMax(w.peaks + 2 * (int64_t)p.batch * p.kv_heads + g, __float_as_uint(lam));
  }
}

// ------------------------------------------------------------------ dK, dV
// Tensor memory: four 64-column buffers, dV at 256, dK_1, dK_2 at 384 and 448.
// Even tiles have S_1, S_2 and G in buffers 0, 1 and 2, odd ones in 3, 2 and 1.
// The threads write W = P_1 - lam P_2 and dS_1 over S_1, dS_2 over S_2, so
//   S_1(i+2) follows the products of W and dS_1(i), which leave its buffer,
//   S_2(i+1) takes the place of G(i) once the threads have read that, and
//   G(i+1) that of dS_2(i), whose product is the first of its tile:
// the scores of the next tile are there when a warp is done with this one, and
// G after the exponentials.  (With both scores issued when G had been read, the
// warps waited 450 to 900 clocks a tile for them: 2800 a tile, now 2300.)  One thread
// issues everything, so a buffer that an earlier product reads may be the target
// of a later one: products run in the order of their issue.  That is what is
// observed, and common in such kernels; the PTX document states it for products
// of one accumulator and shape, which these are not.
template <typename T, int NV>
__device__ __forceinline__ void dkv_cta(const CUtensorMap& mQ, const CUtensorMap& mK, const CUtensorMap& mV,
                                        const CUtensorMap& mG, const amc_diff_attention& p, const DiffBwdWork& wk,
                                        int share) {
  using L = KvSmem<NV>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char diff_sm_raw[];
  unsigned char* sm = (unsigned char*)(((uintptr_t)diff_sm_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* kv_full = (uint64_t*)(sm + L::bar);
  uint64_t* f_full = kv_full + 1;            // [kStages] Q, dO and row pairs landed
  uint64_t* f_empty = f_full + kStages;      // [kStages] their products are done and the pairs read
  uint64_t* s1_full = f_empty + kStages;     // [2] S_1(i) complete, even and odd i
  uint64_t* s2_full = s1_full + 2;           // S_2(i) complete
  uint64_t* g_full = s1_full + 3;            // G(i) complete
  uint64_t* g_read = s1_full + 4;            // the threads have read G(i) (16 warps)
  uint64_t* p_full = s1_full + 5;            // operands of tile i written (16 warps)
  uint64_t* acc_full = s1_full + 6;
  uint32_t* tslot = (uint32_t*)(sm + L::bar + 192);
  volatile int* abort_flag = (volatile int*)(sm + L::bar + 196);
  const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
  // key tiles of one head are launched first tile first: with a causal mask
  // those have the most rows
  const int per = p.kv_heads * p.batch, group = p.heads / p.kv_heads;
  const int unit = blockIdx.x / share, rank = blockIdx.x % share;   // share: CTAs of a cluster
  const int k0 = unit / per * 128, g = unit % per % p.kv_heads, b = unit % per / p.kv_heads;
  const int head0 = g * group + rank * (group / share);
  const DiffLens len = diff_lens(p, b);
  const int first = diff_first_row(len, p.causal, k0) / 64 * 64;
  const int nth = first < len.nq ? (len.nq - first + 63) / 64 : 0;   // tiles a head
  const int nt = (int)warp_uniform(nth * (group / share));
  // pairs behind the tensor's rows are never loaded: they count as zeros
  for (int i = tid; i < kStages * 64; i += kThreadsB)
    reinterpret_cast<float4*>(sm + L::r)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  fence_proxy_async();
  if (tid == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&f_full[i], 1);
      mbar_init(&f_empty[i], 1 + kRowWarps);
    }
    for (int i = 0; i < 3; ++i) mbar_init(&s1_full[i], 1);
    mbar_init(g_full, 1);
    mbar_init(g_read, kRowWarps);
    mbar_init(p_full, kRowWarps);
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (warp == 0) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tslot);
  const uint32_t t_dv = tmem + 256, t_dk = tmem + 384;
  // what the sums of dS and of P_1 - lam P_2 are multiplied with, and the latter's scale over the former's
  float f_dk = p.scale, f_dv = 1.f, to_w = 1.f;
  if constexpr (!kBf16) {
    const DiffShift up = diff_shift(p, wk, b, g);
    f_dk *= diff_pow2(-up.ds);
    f_dv = diff_pow2(-up.w);
    to_w = diff_pow2(up.w - up.ds);
  }
  float* part = (float*)sm;   // [128 keys][kPartPitch] once all products are done

  if (warp == 16) {
    if (lane == 0 && nt > 0) {
      mbar_expect_tx(kv_full, 32768 + NV / 64 * 16384);
      for (int r = 0; r < 128; r += 64) {
        for (int m = 0; m < 2; ++m) tma_load_4d(sm + L::k + m * 16384 + r * 128, &mK, 0, k0 + r, 2 * g + m, b, kv_full);
        for (int c = 0; c < NV / 64; ++c) tma_load_4d(sm + L::v + c * 16384 + r * 128, &mV, 64 * c, k0 + r, g, b, kv_full);
      }
      int h = head0, r0 = first;
      for (int i = 0; i < nt; ++i) {
        const int s = i % kStages;
        if (i >= kStages && !mbar_wait(&f_empty[s], (uint32_t)(i / kStages - 1) & 1u)) { *abort_flag = 1; break; }
        if (*abort_flag) break;
        const int rows = min(64, wk.pitch - r0);
        unsigned char* st = sm + L::f + s * L::stage;
        mbar_expect_tx(&f_full[s], L::stage + rows * 16);
        for (int m = 0; m < 2; ++m) tma_load_4d(st + m * 8192, &mQ, 0, r0, 2 * h + m, b, &f_full[s]);
        for (int c = 0; c < NV / 64; ++c) tma_load_4d(st + 16384 + c * 8192, &mG, 64 * c, r0, h, b, &f_full[s]);
        const int64_t at = (((int64_t)b * p.heads + h) * wk.pitch + r0) / 2;
        bulk_load_1d(sm + L::r + s * 1024, wk.nlse + at, rows * 8, &f_full[s]);
        bulk_load_1d(sm + L::r + s * 1024 + 512, wk.nsum + at, rows * 8, &f_full[s]);
        r0 += 64;
        if (r0 >= len.nq) {
          r0 = first;
          ++h;
        }
      }
    }
  } else if (warp == 17) {
    if (nt > 0) {
      const uint32_t id = idesc_f16(128, 64, kBf16, false, false);
      const uint32_t id_dk = idesc_f16(128, 64, kBf16, false, true);
      const uint32_t id_dv = idesc_f16(128, NV, kBf16, false, true);
      const uint64_t kd = sdesc(smem_addr(sm + L::k), 16, 1024), vd = sdesc(smem_addr(sm + L::v), 16, 1024);
      const uint64_t fd = sdesc(smem_addr(sm + L::f), 16, 1024), fmn = sdesc_mn16(smem_addr(sm + L::f), 8192);
      auto issue_s = [&](int i, int m) {
        const uint64_t st = desc_add(fd, (i % kStages) * L::stage + m * 8192);
        const uint32_t to = tmem + 64 * (m ? 1 + (i & 1) : 3 * (i & 1));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16(to, desc_add(kd, m * 16384 + k * 32), desc_add(st, k * 32), id, k > 0);
        mma_commit_warp(m ? s2_full : &s1_full[i & 1]);
      };
      auto issue_g = [&](int i) {
        const uint64_t st = desc_add(fd, (i % kStages) * L::stage + 16384);
#pragma unroll
        for (int k = 0; k < NV / 16; ++k)
          mma_f16(tmem + 64 * (2 - (i & 1)), desc_add(vd, (k >> 2) * 16384 + (k & 3) * 32),
                  desc_add(st, (k >> 2) * 8192 + (k & 3) * 32), id, k > 0);
        mma_commit_warp(g_full);
      };
      // A operands: warpgroup k wrote rows 16 k .. 16 k + 15 of the tile (K
      // step k) at columns 16 k (+8 for dS_1) of the buffers
      auto issue_dk2 = [&](int i) {
        const uint64_t st = desc_add(fmn, (i % kStages) * L::stage + 8192);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16_ts(t_dk + 64, tmem + 64 * (1 + (i & 1)) + k * 16, desc_add(st, k * 2048), id_dk, i > 0 || k > 0);
      };
      auto issue_acc = [&](int i) {
        const uint64_t st = desc_add(fmn, (i % kStages) * L::stage);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a = tmem + 192 * (i & 1) + k * 16;
          mma_f16_ts(t_dv, a, desc_add(st, 16384 + k * 2048), id_dv, i > 0 || k > 0);
          mma_f16_ts(t_dk, a + 8, desc_add(st, k * 2048), id_dk, i > 0 || k > 0);
        }
        mma_commit_warp(&f_empty[i % kStages]);
      };
      auto landed = [&](int i) { return warp_wait(&f_full[i % kStages], (uint32_t)(i / kStages) & 1u); };
      bool ok = warp_wait(kv_full, 0) && landed(0);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        issue_s(0, 1);
        issue_g(0);
        if (nt > 1 && (ok = landed(1))) issue_s(1, 0);
      }
      for (int i = 0; i < nt && ok; ++i) {
        const bool more = i + 1 < nt;
        if (more) {
          if (!warp_wait(g_read, (uint32_t)i & 1u)) { ok = false; break; }
          tc_fence_after();
          issue_s(i + 1, 1);
        }
        if (!warp_wait(p_full, (uint32_t)i & 1u) || warp_uniform(*abort_flag)) { ok = false; break; }
        tc_fence_after();
        issue_dk2(i);
        if (more) issue_g(i + 1);
        issue_acc(i);
        if (i + 2 < nt) {
          if (!landed(i + 2)) { ok = false; break; }
          issue_s(i + 2, 0);
        }
      }
      if (ok) mma_commit_warp(acc_full);
      else *abort_flag = 1;
    }
  } else {
    // one thread per key; warpgroup w takes rows 16 w .. 16 w + 15 of a tile
    const int w = warp >> 2, t = tid & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const float c2 = p.scale * kLog2e;
    const int fr = diff_first_row(len, p.causal, k0 + t);
    const int fr_all = diff_first_row(len, p.causal, k0 + 127);   // from here on every key of the tile is seen
    const float2 cc = make_float2(c2, c2);
    bool ok = true;
    int h = head0, r0 = first;
    float nlam = nt > 0 ? -wk.lam[h] : 0.f;
    const float2 rw = make_float2(to_w, to_w);
    if (nt > 0) ok = __all_sync(0xffffffffu, mbar_wait(&f_full[0], 0));
    for (int i = 0; i < nt && ok; ++i) {
      const int s = i % kStages;
      const uint32_t x = tmem + lane_base + 16 * w;
      const uint32_t x1 = x + 192 * (i & 1), x2 = x + 64 * (1 + (i & 1)), xg = x + 64 * (2 - (i & 1));
      // The row pairs come from shared memory, whose port the products'
      // operands keep busy: they are read before each wait, not after it.
      const float4* le = reinterpret_cast<const float4*>(sm + L::r + s * 1024 + 128 * w);
      float4 rp[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) rp[j] = le[j];
      ok = __all_sync(0xffffffffu, mbar_wait(&s1_full[i & 1], (uint32_t)(i >> 1) & 1u));
      if (!ok) break;
      tc_fence_after();
      // P_1 and -lam P_2, two rows at a time
      uint32_t sc[16];
      float2 p1[8], p2[8];
      tmem_ld16_nowait(x1, sc);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 a = fma2(make_float2(__uint_as_float(sc[2 * j]), __uint_as_float(sc[2 * j + 1])), cc, make_float2(rp[j].x, rp[j].y));
        p1[j] = make_float2(ex2_approx(a.x), ex2_approx(a.y));
      }
      ok = __all_sync(0xffffffffu, mbar_wait(s2_full, (uint32_t)i & 1u));
      if (!ok) break;
      tc_fence_after();
      tmem_ld16_nowait(x2, sc);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 c = fma2(make_float2(__uint_as_float(sc[2 * j]), __uint_as_float(sc[2 * j + 1])), cc, make_float2(rp[j].z, rp[j].w));
        p2[j] = mul2(make_float2(ex2_approx(c.x), ex2_approx(c.y)), make_float2(nlam, nlam));
      }
      const bool masked = r0 < fr_all || r0 + 64 > len.nq;
      if (masked) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = r0 + 16 * w + 2 * j;
          if (r < fr || r >= len.nq) p1[j].x = p2[j].x = 0.f;
          if (r + 1 < fr || r + 1 >= len.nq) p1[j].y = p2[j].y = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) rp[j] = le[32 + j];
      // the next tile's row pairs, off the path from its scores to its products
      const int sn = (i + 1) % kStages;
      ok = __all_sync(0xffffffffu, (i + 1 == nt || mbar_wait(&f_full[sn], (uint32_t)((i + 1) / kStages) & 1u)) &&
                                       mbar_wait(g_full, (uint32_t)i & 1u));
      if (!ok) break;
      tc_fence_after();
      uint32_t gv[16];
      tmem_ld16_nowait(xg, gv);
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(g_read);
      if (masked) {
        // the values of rows that see nothing may be anything, and 0 times
        // that is not 0
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int r = r0 + 16 * w + j;
          if (r < fr || r >= len.nq) gv[j] = 0u;
        }
        // Q_1, Q_2 and the halves of dO: 8 KB each
        if (r0 + 64 > len.nq && t < 64 && r0 + t >= len.nq && (NV == 128 || w < 3))
          zero_row(sm + L::f + s * L::stage + w * 8192 + t * 128);
        fence_proxy_async();
      }
      float v[8], v1[8], v2[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 d = rp[j];
        const float2 gg = make_float2(__uint_as_float(gv[2 * j]), __uint_as_float(gv[2 * j + 1]));
        float2 both = add2(p1[j], p2[j]);
        if constexpr (!kBf16) both = mul2(both, rw);
        const float2 a = mul2(p1[j], add2(gg, make_float2(d.x, d.y))), c = mul2(p2[j], add2(gg, make_float2(d.z, d.w)));
        v[j] = __uint_as_float(pack2<T>(both.x, both.y));
        v1[j] = __uint_as_float(pack2<T>(a.x, a.y));
        v2[j] = __uint_as_float(pack2<T>(c.x, c.y));
      }
      tmem_st8(x1, v);
      tmem_st8(x1 + 8, v1);
      tmem_st8(x2, v2);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(p_full);
      warp_arrive(&f_empty[s]);
      r0 += 64;
      if (r0 >= len.nq) {
        r0 = first;
        ++h;
        if (i + 1 < nt) nlam = -wk.lam[h];
      }
    }
    if (nt > 0) ok = ok && mbar_wait(acc_full, 0);
    ok = named_bar_and(1, kRowThreads, ok && !*abort_flag);
    if (ok) {
      // warpgroups 0 and 1 write dK_1 and dK_2, 2 and 3 the halves of dV
      tc_fence_after();
      const int key = k0 + t;
      T* dst = w < 2 ? (T*)p.dk + b * p.dks[0] + (2 * g + w) * p.dks[1] + (int64_t)key * p.dks[2]
                     : (T*)p.dv_ + b * p.dvs[0] + g * p.dvs[1] + (int64_t)key * p.dvs[2] + 64 * (w - 2);
      const uint32_t src = (w < 2 ? t_dk + 64 * w : t_dv + 64 * (w - 2)) + lane_base;
      const int cols = w < 2 ? p.d : p.dv - 64 * (w - 2);
      const float f = w < 2 ? f_dk : f_dv;
      if (NV == 128 || w < 3) {
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          float v[16];
          if (nt > 0) tmem_ld16(src + c, v);
          else
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.f;
          if (share > 1) {   // all products are done: the tiles' memory is free
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(part + t * kPartPitch + 64 * w + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else if (key < p.nk && c < cols) {
            store16<T>(dst + c, v, f, cols - c);
          }
        }
      }
    } else if (tid == 0) {
      *abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (tid == 0) atomicExch(&g_diff_bwd_error, AMC_ERR_TIMEOUT);
    // bounded drain of copies and products still in flight
    mbar_wait(kv_full, 0, 1 << 14);
    for (int i = 0; i < kStages; ++i) mbar_wait(&f_full[i], 0, 1 << 14);
    for (int i = 0; i < 3; ++i) mbar_wait(&s1_full[i], 0, 1 << 14);
    mbar_wait(g_full, 0, 1 << 14);
    mbar_wait(acc_full, 0, 1 << 14);
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc(tmem, 512);
  if (share > 1) {
    // every CTA of the cluster adds up its part of the 128 keys: 4 columns of
    // dK_1, dK_2 and dV a thread, ranks in order
    cluster_sync();
    const int keys = (128 + share - 1) / share;
    for (int i = tid; i < keys * 64; i += kThreadsB) {
      const int row = rank * keys + i / 64, c = i % 64 * 4, key = k0 + row;
      if (row >= 128 || key >= p.nk || (NV == 64 && c >= 192)) continue;
      float4 sum = ld_cluster(part + row * kPartPitch + c, 0);
      for (int r = 1; r < share; ++r) {
        const float4 v = ld_cluster(part + row * kPartPitch + c, r);
        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
      }
      const int m = c / 64, cc = m < 2 ? c % 64 : c - 128;
      if (cc >= (m < 2 ? p.d : p.dv)) continue;
      const float f = m < 2 ? f_dk : f_dv;
      T* dst = m < 2 ? (T*)p.dk + b * p.dks[0] + (2 * g + m) * p.dks[1] + (int64_t)key * p.dks[2]
                     : (T*)p.dv_ + b * p.dvs[0] + g * p.dvs[1] + (int64_t)key * p.dvs[2];
      *reinterpret_cast<uint2*>(dst + cc) = make_uint2(pack2<T>(sum.x * f, sum.y * f), pack2<T>(sum.z * f, sum.w * f));
    }
    cluster_sync();   // the others have read this CTA's part
  }
}

// ------------------------------------------------------------------ dQ, dlam
// Tensor memory: two buffers of S_1, S_2, G (64 columns each) at 0 and 192,
// dQ_1, dQ_2 at 384 and 448.  Tile j+2 is computed into the buffer of tile j
// right after the products that read dS(j) from it (in the order of issue, as
// above), while the threads work on tile j+1.
template <typename T, int NV>
__device__ __forceinline__ void dq_cta(const CUtensorMap& mQ, const CUtensorMap& mK, const CUtensorMap& mV,
                                       const CUtensorMap& mG, const amc_diff_attention& p, const DiffBwdWork& wk,
                                       int index) {
  using L = QSmem<NV>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char diff_sm_raw[];
  unsigned char* sm = (unsigned char*)(((uintptr_t)diff_sm_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* q_full = (uint64_t*)(sm + L::bar);
  uint64_t* f_full = q_full + 1;             // [kStages]
  uint64_t* f_empty = f_full + kStages;      // [kStages]
  uint64_t* s_full = f_empty + kStages;      // [2] S_1, S_2, G of a buffer
  uint64_t* p_full = s_full + 2;             // [2] dS written (16 warps)
  uint64_t* acc_full = p_full + 2;
  uint32_t* tslot = (uint32_t*)(sm + L::bar + 192);
  volatile int* abort_flag = (volatile int*)(sm + L::bar + 196);
  float* red = (float*)(sm + L::bar + 256);  // [16]
  const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
  const int per = p.heads * p.batch, tiles = (p.nq + 127) / 128;
  const int tile = tiles - 1 - index / per, h = index % per % p.heads, b = index % per / p.heads;
  const int g = h / (p.heads / p.kv_heads), r0 = tile * 128;
  const DiffLens len = diff_lens(p, b);
  const int last = min(r0 + 128, len.nq) - 1;
  const int kend = last >= r0 ? diff_limit(len, p.causal, last) : 0;
  const int nt = (int)warp_uniform((kend + 63) / 64);
  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&f_full[i], 1);
      mbar_init(&f_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kRowWarps);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (warp == 0) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tslot);
  const uint32_t t_dq = tmem + 384;
  float back = 1.f;   // P carries the scale of dS
  if constexpr (!kBf16) back = diff_pow2(-diff_shift(p, wk, b, g).ds);

  if (warp == 16) {
    if (lane == 0 && nt > 0) {
      mbar_expect_tx(q_full, 32768 + NV / 64 * 16384);
      for (int r = 0; r < 128; r += 64) {
        for (int m = 0; m < 2; ++m) tma_load_4d(sm + L::q + m * 16384 + r * 128, &mQ, 0, r0 + r, 2 * h + m, b, q_full);
        for (int c = 0; c < NV / 64; ++c) tma_load_4d(sm + L::g + c * 16384 + r * 128, &mG, 64 * c, r0 + r, h, b, q_full);
      }
      for (int j = 0; j < nt; ++j) {
        const int s = j % kStages;
        if (j >= kStages && !mbar_wait(&f_empty[s], (uint32_t)(j / kStages - 1) & 1u)) { *abort_flag = 1; break; }
        if (*abort_flag) break;
        unsigned char* st = sm + L::f + s * L::stage;
        mbar_expect_tx(&f_full[s], L::stage);
        for (int m = 0; m < 2; ++m) tma_load_4d(st + m * 8192, &mK, 0, j * 64, 2 * g + m, b, &f_full[s]);
        for (int c = 0; c < NV / 64; ++c) tma_load_4d(st + 16384 + c * 8192, &mV, 64 * c, j * 64, g, b, &f_full[s]);
      }
    }
  } else if (warp == 17) {
    if (nt > 0) {
      const uint32_t id = idesc_f16(128, 64, kBf16, false, false);
      const uint32_t id_dq = idesc_f16(128, 64, kBf16, false, true);
      const uint64_t qd = sdesc(smem_addr(sm + L::q), 16, 1024), gd = sdesc(smem_addr(sm + L::g), 16, 1024);
      const uint64_t fd = sdesc(smem_addr(sm + L::f), 16, 1024), fmn = sdesc_mn16(smem_addr(sm + L::f), 8192);
      auto issue_s = [&](int j) -> bool {
        if (!warp_wait(&f_full[j % kStages], (uint32_t)(j / kStages) & 1u)) return false;
        tc_fence_after();
        const uint64_t st = desc_add(fd, (j % kStages) * L::stage);
        const uint32_t x = tmem + (j & 1) * 192;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16(x + m * 64, desc_add(qd, m * 16384 + k * 32), desc_add(st, m * 8192 + k * 32), id, k > 0);
#pragma unroll
        for (int k = 0; k < NV / 16; ++k)
          mma_f16(x + 128, desc_add(gd, (k >> 2) * 16384 + (k & 3) * 32),
                  desc_add(st, 16384 + (k >> 2) * 8192 + (k & 3) * 32), id, k > 0);
        mma_commit_warp(&s_full[j & 1]);
        return true;
      };
      bool ok = warp_wait(q_full, 0);
      for (int j = 0; j < 2 && j < nt && ok; ++j) ok = issue_s(j);
      for (int j = 0; j < nt && ok; ++j) {
        if (!warp_wait(&p_full[j & 1], (uint32_t)(j >> 1) & 1u) || warp_uniform(*abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint64_t st = desc_add(fmn, (j % kStages) * L::stage);
        const uint32_t x = tmem + (j & 1) * 192;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a = x + k * 16;   // warpgroup k wrote keys 16 k .. of the tile
          mma_f16_ts(t_dq, a, desc_add(st, k * 2048), id_dq, j > 0 || k > 0);
          mma_f16_ts(t_dq + 64, a + 64, desc_add(st, 8192 + k * 2048), id_dq, j > 0 || k > 0);
        }
        mma_commit_warp(&f_empty[j % kStages]);
        if (j + 2 < nt) ok = issue_s(j + 2);
      }
      if (ok) mma_commit_warp(acc_full);
      else *abort_flag = 1;
    }
  } else {
    // one thread per row; warpgroup w takes keys 16 w .. 16 w + 15 of a tile
    const int w = warp >> 2, t = tid & 127, row = r0 + t;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const float c2 = p.scale * kLog2e, lam = wk.lam[h];
    const int lim = diff_limit(len, p.causal, row);
    const int all_see = r0 + 127 < len.nq ? diff_limit(len, p.causal, r0) : 0;
    float2 e = make_float2(-INFINITY, -INFINITY), ds = make_float2(0.f, 0.f);
    if (lim > 0) {
      const int64_t at = ((int64_t)b * p.heads + h) * wk.pitch;
      e = make_float2(diff_row(wk.nlse, at, row, 0), diff_row(wk.nlse, at, row, 1));
      ds = make_float2(diff_row(wk.nsum, at, row, 0), diff_row(wk.nsum, at, row, 1));
    }
    const float2 cc = make_float2(c2, c2), e1 = make_float2(e.x, e.x), e2 = make_float2(e.y, e.y);
    const float2 d1 = make_float2(ds.x, ds.x), d2 = make_float2(ds.y, ds.y), nl = make_float2(-lam, -lam);
    float pg = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      const uint32_t x = tmem + (j & 1) * 192 + lane_base + 16 * w;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[j & 1], (uint32_t)(j >> 1) & 1u));
      if (!ok) break;
      tc_fence_after();
      uint32_t s1[16], s2[16], gv[16];
      tmem_ld16_nowait(x, s1);
      tmem_ld16_nowait(x + 64, s2);
      tmem_ld16_nowait(x + 128, gv);
      tmem_ld_wait();
      if (j * 64 + 64 > all_see) {
        const int n = lim - j * 64 - 16 * w;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i >= n) {
            s1[i] = s2[i] = 0xff800000u;
            gv[i] = 0u;
          }
        // K behind the length may hold anything, and 0 times it is not 0
        if (j * 64 + 64 > len.nk && len.nk < p.nk && w < 2 && t < 64 && j * 64 + t >= len.nk)
          zero_row(sm + L::f + (j % kStages) * L::stage + w * 8192 + t * 128);
        fence_proxy_async();
      }
      float2 part[2] = {};
      float v1[8], v2[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 gg = make_float2(__uint_as_float(gv[2 * i]), __uint_as_float(gv[2 * i + 1]));
        const float2 a = fma2(make_float2(__uint_as_float(s1[2 * i]), __uint_as_float(s1[2 * i + 1])), cc, e1);
        const float2 c = fma2(make_float2(__uint_as_float(s2[2 * i]), __uint_as_float(s2[2 * i + 1])), cc, e2);
        const float2 p1 = make_float2(ex2_approx(a.x), ex2_approx(a.y)), p2 = make_float2(ex2_approx(c.x), ex2_approx(c.y));
        part[i & 1] = fma2(p2, gg, part[i & 1]);
        const float2 q1 = mul2(p1, add2(gg, d1)), q2 = mul2(mul2(p2, nl), add2(gg, d2));
        v1[i] = __uint_as_float(pack2<T>(q1.x, q1.y));
        v2[i] = __uint_as_float(pack2<T>(q2.x, q2.y));
      }
      tmem_st8(x, v1);
      tmem_st8(x + 64, v2);
      tmem_st_wait();
      pg += (part[0].x + part[0].y) + (part[1].x + part[1].y);
      tc_fence_before();
      warp_arrive(&p_full[j & 1]);
    }
    if (nt > 0) ok = ok && mbar_wait(acc_full, 0);
    for (int o = 16; o > 0; o >>= 1) pg += __shfl_xor_sync(0xffffffffu, pg, o);
    if (lane == 0) red[warp] = pg;
    ok = named_bar_and(1, kRowThreads, ok && !*abort_flag);
    if (ok) {
      tc_fence_after();
      // warpgroup w writes 32 columns of dQ_1 (w = 0, 1) or dQ_2
      const int m = w >> 1, c0 = 32 * (w & 1);
      T* dq = (T*)p.dq + b * p.dqs[0] + (2 * h + m) * p.dqs[1] + (int64_t)row * p.dqs[2];
#pragma unroll 1
      for (int c = c0; c < c0 + 32; c += 16) {
        float v[16];
        if (nt > 0) tmem_ld16(t_dq + 64 * m + lane_base + c, v);
        else
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0.f;
        if (row < p.nq && c < p.d) store16<T>(dq + c, v, p.scale * back, p.d - c);
      }
      if (tid == 0) {
        float sum = 0.f;
        for (int i = 0; i < kRowWarps; ++i) sum += red[i];
        wk.partials[((int64_t)h * p.batch + b) * tiles + tile] = sum * back;
      }
    } else if (tid == 0) {
      *abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (tid == 0) atomicExch(&g_diff_bwd_error, AMC_ERR_TIMEOUT);
    mbar_wait(q_full, 0, 1 << 14);
    for (int i = 0; i < kStages; ++i) mbar_wait(&f_full[i], 0, 1 << 14);
    for (int i = 0; i < 2; ++i) mbar_wait(&s_full[i], 0, 1 << 14);
    mbar_wait(acc_full, 0, 1 << 14);
  }
  if (warp == 0) tmem_dealloc(tmem, 512);
  diff_dlam_last<T>(p, wk, h, tiles, reinterpret_cast<double*>(sm));   // all products are done
}

template <typename T, int NV>
__global__ void __launch_bounds__(kThreadsB, 1) k_diff_bwd_tc(
    const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mK,
    const __grid_constant__ CUtensorMap mV, const __grid_constant__ CUtensorMap mG,
    const __grid_constant__ amc_diff_attention p, const __grid_constant__ DiffBwdWork wk, int dkv_ctas, int dq_ctas,
    int share) {
  if ((int)blockIdx.x < dkv_ctas) dkv_cta<T, NV>(mQ, mK, mV, mG, p, wk, share);
  else if ((int)blockIdx.x - dkv_ctas < dq_ctas) dq_cta<T, NV>(mQ, mK, mV, mG, p, wk, (int)blockIdx.x - dkv_ctas);
}

namespace {

bool aligned_out(const void* x, const int64_t s[3], int64_t heads, int64_t rows, int64_t batch) {
  return !((uintptr_t)x & 15) && (batch == 1 || s[0] % 8 == 0) && (heads == 1 || s[1] % 8 == 0) &&
         (rows == 1 || s[2] % 8 == 0);
}

template <typename T, int NV>
int bwd_tc(const amc_diff_attention& p, const DiffBwdWork& w, const CUtensorMap (&map)[4], cudaStream_t s) {
  static std::atomic<uint64_t> once{0};
  constexpr int bytes = KvSmem<NV>::bytes > QSmem<NV>::bytes ? KvSmem<NV>::bytes : QSmem<NV>::bytes;
  if (int rc = smem_attr_once(k_diff_bwd_tc<T, NV>, bytes, once)) return rc;
  const int64_t units = (int64_t)((p.nk + 127) / 128) * p.kv_heads * p.batch;
  const int share = diff_share(p, units);
  const int64_t dq = (int64_t)((p.nq + 127) / 128) * p.heads * p.batch;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * share + (dq + share - 1) / share * share));
  cfg.blockDim = dim3(kThreadsB);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)share, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = share > 1 ? 1 : 0;
  AMC_CUDA(cudaLaunchKernelEx(&cfg, k_diff_bwd_tc<T, NV>, map[0], map[1], map[2], map[3], p, w, (int)(units * share),
                              (int)dq, share));
  return AMC_OK;
}

}  // namespace

int diff_bwd_tc(const amc_diff_attention& p, const DiffBwdWork& w, cudaStream_t s, bool* handled) {
  *handled = false;
  if (!diff_tc_shape(p) || p.nq <= 0 || !(p.scale > 0.f)) return AMC_OK;   // masked scores are -inf before the scale
  if (!aligned_out(p.dq, p.dqs, 2 * p.heads, p.nq, p.batch) || !aligned_out(p.dk, p.dks, 2 * p.kv_heads, p.nk, p.batch) ||
      !aligned_out(p.dv_, p.dvs, p.kv_heads, p.nk, p.batch))
    return AMC_OK;
  if ((int64_t)((p.nq + 127) / 128) * p.heads * p.batch + (int64_t)((p.nk + 127) / 128) * p.kv_heads * p.batch > 0x7ffffff0)
    return AMC_OK;
  const bool bf16 = p.dtype == AMC_BF16;
  CUtensorMap map[4];   // boxes of 64 rows
  int rc = make_tmap_4d_16(&map[0], p.q, bf16, p.batch, 2 * p.heads, p.nq, p.d, p.qs, 64);
  if (!rc) rc = make_tmap_4d_16(&map[1], p.k, bf16, p.batch, 2 * p.kv_heads, p.nk, p.d, p.ks, 64);
  if (!rc) rc = make_tmap_4d_16(&map[2], p.v, bf16, p.batch, p.kv_heads, p.nk, p.dv, p.vs, 64);
  if (!rc) rc = make_tmap_4d_16(&map[3], p.d_o, bf16, p.batch, p.heads, p.nq, p.dv, p.dos, 64);
  if (rc == AMC_ERR_UNSUPPORTED) return AMC_OK;
  if (rc) return rc;
  *handled = true;
  if (!bf16) {
    AMC_CUDA(cudaMemsetAsync(w.peaks, 0, diff_peaks(p) * sizeof(unsigned), s));
    const int rows = p.nq > p.nk ? p.nq : p.nk;
    k_diff_peaks<<<dim3((rows + kPeakRows - 1) / kPeakRows, p.heads + p.kv_heads, p.batch), 256, 0, s>>>(p, w);
    AMC_CUDA(cudaGetLastError());
  }
  if ((rc = launch_diff_bwd_rows(p, w, s))) return rc;
  if (bf16) return p.dv <= 64 ? bwd_tc<__nv_bfloat16, 64>(p, w, map, s) : bwd_tc<__nv_bfloat16, 128>(p, w, map, s);
  return p.dv <= 64 ? bwd_tc<__half, 64>(p, w, map, s) : bwd_tc<__half, 128>(p, w, map, s);
}

int diff_bwd_check_error() {
  int e = 0;
  AMC_CUDA(cudaMemcpyFromSymbol(&e, g_diff_bwd_error, sizeof(int)));
  if (e) {
    int z = 0;
    AMC_CUDA(cudaMemcpyToSymbol(g_diff_bwd_error, &z, sizeof(int)));
    return fail(e, "diff_attention backward: a bounded wait on the tensor-core pipeline gave up");
  }
  return AMC_OK;
}

}  // namespace amc
