// Differential attention forward on the tensor cores (sm_100a, tcgen05
// kind::f16), 16-bit tensors with d <= 64 and dv <= 128, both multiples of 8.
//
// A CTA owns 128 query rows of one head.  Its two maps are two warpgroups,
// one thread per row, that share the V tile; 128-key tiles stream through
// shared memory by TMA (smaller heads are zero-filled to 64 / NV columns) and
// are worked off in steps of 64 keys.  Warp 8 loads; warps 9 and 10 issue, a map
// each.
// Tensor memory holds two 64-column score buffers per map and O_0, O_1 (NV
// columns each): all 512 columns at NV = 128, which is why one CTA takes
// exactly one tile of both maps.  P(j) goes back over its own scores as
// 16-bit pairs and is the A operand of P V from there (V MN-major, as TMA
// wrote it); S(j+2) follows P(j) V into the same buffer.  So while a group is
// in the softmax of step j, its products of j-1 and the scores of j+1 run, and
// neither group waits for the other.  (With one 128-column buffer a map, both
// groups' exponentials met and the pipes took turns: 3550 clocks a tile.)
//   p = 2^(scale log2e s - m), rounded to the tensors' type for P V and
//   summed unrounded; m follows the row maximum only when it rises by more
//   than 2^8 (a rule known from published attention kernels; any bound is right
//   that leaves 2^bound times a sum of weights in range), and O is rescaled then,
//   once P V of the step before is complete.
// P's rounding, half a step of the type for each weight, is the price of feeding
// it to the tensor pipe: o is 1.5 times as far from 64 bits as from f32 products
// rounded once (0.0025 against 0.0017 of its norm in bf16).
// That S(j+2) may follow P(j) V into the buffer that holds P(j) without a wait rests
// on one thread's products running in the order of their issue, which is observed;
// the PTX document states it for products of one accumulator and shape.
// The two rows' results meet in the epilogue: O = O_0 / l_0 - lam O_1 / l_1.
//
// Bound: per 128 x 128 tile of both maps the products take 1536 clocks of the
// tensor pipe, their operands 1800 of the shared-memory port, and the 32768
// exponentials 2048 of the special-function unit.  Taking a part of those on
// the FMA pipe by a polynomial gained nothing: the softmax threads' other
// instructions then fill the time.
// Measured: 4096 x 4096, causal, 16 heads (4 key heads), 4 sequences, d 64: 446 us
// in a short run, 496 in a long one (412 GFLOP: 924 and 831 TFLOP/s); 333 rows that
// continue 777 keys, causal, 8 heads, 6 sequences of mixed lengths, d 64: 21 us;
// 1000 x 1000, causal, 6 heads, 5 sequences of mixed lengths, d 48: 27 us.
// Every wait is bounded; on expiry the kernel records AMC_ERR_TIMEOUT and
// leaves after its copies and products have drained.
#include <cmath>
#include <type_traits>

#include "amc_diffattn.h"
#include "amc_half.cuh"
#include "amc_tc.cuh"

namespace amc {

using namespace tc;

namespace {

constexpr int kThreadsF = 352;      // warps 0-7 softmax, 8 loads, 9 and 10 issue
constexpr int kKStages = 3, kVStages = 2;
constexpr float kLog2e = 1.4426950408889634f;

template <int NV>
struct FwdSmem {
  static constexpr int q = 0;                              // 2 maps x 16 KB
  static constexpr int k = 32768;                          // stages x 2 maps x 16 KB
  static constexpr int v = k + kKStages * 32768;           // stages x NV/64 x 16 KB
  static constexpr int v_bytes = NV / 64 * 16384;
  static constexpr int x = v + kVStages * v_bytes;         // 2 x 128 row factors
  static constexpr int bar = x + 1024;
  static constexpr int bytes = bar + 256 + 1024;
};

__device__ int g_diff_error;

}  // namespace

template <typename T, int NV>
__global__ void __launch_bounds__(kThreadsF, 1) k_diff_fwd_tc(const __grid_constant__ CUtensorMap mQ,
                                                             const __grid_constant__ CUtensorMap mK,
                                                             const __grid_constant__ CUtensorMap mV,
                                                             const __grid_constant__ amc_diff_attention p) {
  using L = FwdSmem<NV>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char diff_sm_raw[];
  unsigned char* sm = (unsigned char*)(((uintptr_t)diff_sm_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* q_full = (uint64_t*)(sm + L::bar);
  uint64_t* k_full = q_full + 1;                  // [kKStages]
  uint64_t* k_empty = k_full + kKStages;
  uint64_t* v_full = k_empty + kKStages;          // [kVStages]
  uint64_t* v_empty = v_full + kVStages;
  uint64_t* s_full = v_empty + kVStages;          // [map][buffer] S(j) complete
  uint64_t* p_full = s_full + 4;                  // [map][buffer] P(j) written (4 warps)
  uint64_t* o_done = p_full + 4;                  // [map] P V of a step complete
  uint64_t* all_done = o_done + 2;
  uint32_t* tslot = (uint32_t*)(sm + L::bar + 192);
  volatile int* abort_flag = (volatile int*)(sm + L::bar + 196);
  const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
  // Tiles of one head are launched last row tile first (with a causal mask
  // those see the most keys), the heads of one key head next to each other.
  const int per = p.heads * p.batch, tiles = (p.nq + 127) / 128;
  const int tile = tiles - 1 - (int)(blockIdx.x / per), h = blockIdx.x % per % p.heads, b = blockIdx.x % per / p.heads;
  const int g = h / (p.heads / p.kv_heads), r0 = tile * 128;
  const DiffLens len = diff_lens(p, b);
  const int last = min(r0 + 128, len.nq) - 1;
  const int kend = last >= r0 ? diff_limit(len, p.causal, last) : 0;
  const int nt = (int)warp_uniform((kend + 127) / 128), ns = (int)warp_uniform((kend + 63) / 64);
  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kKStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
    }
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(&o_done[0], 1);
    mbar_init(&o_done[1], 1);
    mbar_init(all_done, 2);
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (warp == 0) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tslot);   // S_m at 128 m + 64 (j & 1), O_m at 256 + 128 m

  if (warp == 8) {
    if (lane == 0 && nt > 0) {
      mbar_expect_tx(q_full, 32768);
      for (int m = 0; m < 2; ++m) tma_load_4d(sm + L::q + m * 16384, &mQ, 0, r0, 2 * h + m, b, q_full);
      for (int j = 0; j < nt; ++j) {
        const int s = j % kKStages, t = j % kVStages;
        if (j >= kKStages && !mbar_wait(&k_empty[s], (uint32_t)(j / kKStages - 1) & 1u)) { *abort_flag = 1; break; }
        mbar_expect_tx(&k_full[s], 32768);
        for (int m = 0; m < 2; ++m)
          tma_load_4d(sm + L::k + s * 32768 + m * 16384, &mK, 0, j * 128, 2 * g + m, b, &k_full[s]);
        if (j >= kVStages && !mbar_wait(&v_empty[t], (uint32_t)(j / kVStages - 1) & 1u)) { *abort_flag = 1; break; }
        if (*abort_flag) break;
        mbar_expect_tx(&v_full[t], L::v_bytes);
        for (int c = 0; c < NV / 64; ++c)
          tma_load_4d(sm + L::v + t * L::v_bytes + c * 16384, &mV, 64 * c, j * 128, g, b, &v_full[t]);
      }
    }
  } else if (warp >= 9) {
    if (nt > 0) {
      const int m = warp - 9;
      const uint32_t id_s = idesc_f16(128, 64, kBf16, false, false);
      const uint32_t id_o = idesc_f16(128, NV, kBf16, false, true);
      const uint64_t qd = sdesc(smem_addr(sm + L::q), 16, 1024), kd = sdesc(smem_addr(sm + L::k), 16, 1024);
      const uint64_t vd = sdesc_mn16(smem_addr(sm + L::v), 16384);
      const int ksteps = (p.d + 15) / 16;
      // step j: keys 64 j .. 64 j + 63, half j & 1 of tile j / 2
      auto issue_s = [&](int j) {
        const uint64_t qb = desc_add(qd, m * 16384);
        const uint64_t kb = desc_add(kd, ((j >> 1) % kKStages) * 32768 + m * 16384 + (j & 1) * 8192);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < ksteps)
            mma_f16(tmem + m * 128 + (j & 1) * 64, desc_add(qb, k * 32), desc_add(kb, k * 32), id_s, k > 0);
        mma_commit_warp(&s_full[2 * m + (j & 1)]);
      };
      auto issue_pv = [&](int j) {
        const uint64_t vb = desc_add(vd, ((j >> 1) % kVStages) * L::v_bytes + (j & 1) * 8192);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16_ts(tmem + 256 + m * 128, tmem + m * 128 + (j & 1) * 64 + k * 8, desc_add(vb, k * 2048), id_o,
                     j > 0 || k > 0);
        mma_commit_warp(&o_done[m]);
      };
      bool ok = warp_wait(q_full, 0) && warp_wait(&k_full[0], 0);
      if (ok) {
        tc_fence_after();
        for (int j = 0; j < 2 && j < ns; ++j) issue_s(j);
        mma_commit_warp(&k_empty[0]);
      }
      for (int j = 0; j < ns && ok; ++j) {
        const int tv = j >> 1, tk = (j + 2) >> 1;
        const bool more = j + 2 < ns;
        ok = (j & 1) || warp_wait(&v_full[tv % kVStages], (uint32_t)(tv / kVStages) & 1u);
        if (ok && more && !(j & 1)) ok = warp_wait(&k_full[tk % kKStages], (uint32_t)(tk / kKStages) & 1u);
        ok = ok && warp_wait(&p_full[2 * m + (j & 1)], (uint32_t)(j >> 1) & 1u) && !warp_uniform(*abort_flag);
        if (!ok) break;
        tc_fence_after();
        issue_pv(j);
        if (more) issue_s(j + 2);
        // both halves of a tile are used: its stage may be refilled
        if ((j & 1) || j + 1 == ns) mma_commit_warp(&v_empty[tv % kVStages]);
        if (more && ((j & 1) || j + 3 == ns)) mma_commit_warp(&k_empty[tk % kKStages]);
      }
      if (ok) mma_commit_warp(all_done);
      else *abort_flag = 1;
    }
  } else {
    // ---------------- softmax of map m, one thread per query row
    const int m = warp >> 2, t = tid & 127, row = r0 + t;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + m * 128 + lane_base, t_o = tmem + 256 + m * 128 + lane_base;
    const float c2 = p.scale * kLog2e;
    const int lim = diff_limit(len, p.causal, row);
    // steps that end at or below this need no mask in any row of the CTA
    const int all_see = r0 + 127 < len.nq ? diff_limit(len, p.causal, r0) : 0;
    float top = -INFINITY;
    float2 l2 = make_float2(0.f, 0.f);
    bool ok = true;
    for (int j = 0; j < ns; ++j) {
      const uint32_t t_b = t_s + (j & 1) * 64;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * m + (j & 1)], (uint32_t)(j >> 1) & 1u) && !*abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[2][32];
      tmem_ld32_nowait(t_b, sr[0]);
      tmem_ld32_nowait(t_b + 32, sr[1]);
      tmem_ld_wait();
      const bool masked = j * 64 + 64 > all_see;
      if (masked) {
        const int n = lim - j * 64;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (32 * c + i >= n) sr[c][i] = 0xff800000u;
        if (j * 64 + 64 > len.nk && len.nk < p.nk) {
          // V behind the length may hold anything, and 0 times it is not 0:
          // clear those rows of the step before any product reads them
          const int vs = (j >> 1) % kVStages, r = (j & 1) * 64 + (t & 63);
          ok = __all_sync(0xffffffffu, mbar_wait(&v_full[vs], (uint32_t)((j >> 1) / kVStages) & 1u));
          if (!ok) break;
          if ((j >> 1) * 128 + r >= len.nk && (t >> 6) < NV / 64) {
            unsigned char* vr = sm + L::v + vs * L::v_bytes + (t >> 6) * 16384 + r * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<int4*>(vr + 16 * i) = make_int4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
      const float mt = c2 * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool up = mt > top + 8.f;
      if (__any_sync(0xffffffffu, up)) {
        const float corr = up ? ex2_approx(top - mt) : 1.f;   // 0 at the first key
        if (up) {
          l2 = mul2(l2, make_float2(corr, corr));
          top = mt;
        }
        if (j > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&o_done[m], (uint32_t)(j - 1) & 1u));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < NV; c += 16) {
            float v[16];
            tmem_ld16(t_o + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= corr;
            tmem_st16(t_o + c, v);
          }
        }
      }
      const float base = top == -INFINITY ? 0.f : top;   // a row that has seen no key
      const float2 cc = make_float2(c2, c2), nb = make_float2(-base, -base);
      float2 s4[4] = {};
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 x = fma2(make_float2(__uint_as_float(sr[i >> 4][2 * (i & 15)]),
                                          __uint_as_float(sr[i >> 4][2 * (i & 15) + 1])), cc, nb);
        const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
        s4[i & 3] = add2(s4[i & 3], e);
        v[i] = __uint_as_float(pack2<T>(e.x, e.y));
      }
      tmem_st32(t_b, v);
      tmem_st_wait();
      l2 = add2(l2, add2(add2(s4[0], s4[1]), add2(s4[2], s4[3])));
      tc_fence_before();
      warp_arrive(&p_full[2 * m + (j & 1)]);
    }
    const float l = l2.x + l2.y;
    if (ns > 0) ok = ok && mbar_wait(all_done, 0);
    const float lam = lam_of<T>(p, h);
    float* xch = (float*)(sm + L::x);
    xch[m * 128 + t] = l != 0.f ? 1.f / l : 0.f;
    ok = named_bar_and(1, 256, ok && !*abort_flag);
    if (ok) {
      // warpgroup m writes columns 64 m .. of both results (NV = 64: group 0 alone)
      tc_fence_after();
      if (row < p.nq) {
        if (p.lse) p.lse[((int64_t)b * 2 * p.heads + 2 * h + m) * p.nq + row] =
            row_lse(top, l);
      }
      const float f0 = xch[t], f1 = xch[128 + t], f = -lam;
      if (64 * m < NV) {
        T* o = (T*)p.o + b * p.os[0] + h * p.os[1] + (int64_t)row * p.os[2] + 64 * m;
        T* o2 = p.o2 ? (T*)p.o2 + b * p.o2s[0] + h * p.o2s[1] + (int64_t)row * p.o2s[2] + 64 * m : nullptr;
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          float a0[16], a1[16];
          if (nt > 0) {
            tmem_ld16(tmem + 256 + lane_base + 64 * m + c, a0);
            tmem_ld16(tmem + 384 + lane_base + 64 * m + c, a1);
          }
          uint32_t w[8], w2[8];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            a1[i] = ns > 0 ? a1[i] * f1 : 0.f;
            a0[i] = ns > 0 ? fmaf(f, a1[i], a0[i] * f0) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            w[i] = pack2<T>(a0[2 * i], a0[2 * i + 1]);
            w2[i] = pack2<T>(a1[2 * i], a1[2 * i + 1]);
          }
          if (row < p.nq) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (64 * m + c + 8 * i < p.dv) {
                *reinterpret_cast<uint4*>(o + c + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                if (o2)
                  *reinterpret_cast<uint4*>(o2 + c + 8 * i) = make_uint4(w2[4 * i], w2[4 * i + 1], w2[4 * i + 2], w2[4 * i + 3]);
              }
          }
        }
      }
    } else if (t == 0) {
      *abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (tid == 0) atomicExch(&g_diff_error, AMC_ERR_TIMEOUT);
    // bounded drain of copies and products still in flight
    mbar_wait(q_full, 0, 1 << 14);
    for (int i = 0; i < kKStages; ++i) mbar_wait(&k_full[i], 0, 1 << 14);
    for (int i = 0; i < kVStages; ++i) mbar_wait(&v_full[i], 0, 1 << 14);
    for (int i = 0; i < 4; ++i) mbar_wait(&s_full[i], 0, 1 << 14);
    mbar_wait(all_done, 0, 1 << 14);
  }
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ CTA pairs
// The kernel for many rows over few keys.  One CTA of 128 rows asks the L2 for 512
// bytes a key (d = 64), 7.6 TB/s at 150 clocks a key.  Here two CTAs own 256 rows of
// one head and their products are cta_group::2: each CTA stages half the keys of K (N of the
// scores) and half the columns of V (N of P V), so the traffic per row halves,
// and so do the products to issue.  The CTAs are persistent, one pair per two
// SMs: the next tile's Q, K and V load, and its first scores run, while the
// softmax warps write the last tile's result.
// In each CTA warps 0-7 are the softmax of its 128 rows and two maps, warp 8
// loads its halves and warp 10 passes on that they have landed; warp 9 of the
// even CTA issues.  The issuer paces the pipe: every wait and every commit
// costs it 100 to 200 clocks, so a step of both maps has one barrier each way
// (scores ready, P written), a tile one for all its loads, and P V of the step
// before needs none of its own: the scores after next follow it on the pipe,
// and their barrier is committed even where there is no such step.
// What the odd CTA's shared memory holds (loaded tiles, cleared rows of V) is
// released and acquired at cluster scope; that costs nothing measurable (16 heads
// x 4 sequences, 4096 x 4096, causal: the same with and without it).
// Measured, 8 heads x 16 sequences, 2048 x 2048, d 64, no mask: 466 us in a short
// run, 543 in a long one at the power limit (412 GFLOP: 884 and 759 TFLOP/s), of
// which about a sixth is the turnover from tile to tile (843,727 cycles of the
// kernel, of which the 14 tiles' 32 steps of 1577 are 706,496).  Within a step the
// tensor pipe is busy for 847 clocks and the special-function unit for 1024, and
// issue slots are 38 % taken: the rest are waits for one another.  Staggering the
// two maps by half a step, 16 softmax warps instead of 8, and a part of the
// exponentials on the FMA pipe each made it slower or gained nothing.
namespace {

constexpr int kPStages = 5;

struct PairSmem {
  static constexpr int q = 0;                        // 2 maps x 16 KB
  static constexpr int kv = 32768;                   // stages of one 128-key tile:
  static constexpr int v = 16384;                    //   K [half of the tile][map] 32 keys x 128 B, then V 128 keys x 64 columns
  static constexpr int stage = 32768;
  static constexpr int x = kv + kPStages * stage;    // 2 x 128 row factors
  static constexpr int bar = x + 1024;
  static constexpr int bytes = bar + 256 + 1024;
};

// The next of the tiles that a pair works off: 256 rows of one head.
struct PairItem {
  int b, h, g, r0, kend, nt, ns;
  DiffLens len;
};
__device__ __forceinline__ PairItem pair_item(const amc_diff_attention& p, int w) {
  const int per = p.heads * p.batch, tiles = (p.nq + 255) / 256;
  PairItem t;
  t.h = w % per % p.heads;
  t.b = w % per / p.heads;
  t.g = t.h / (p.heads / p.kv_heads);
  t.r0 = (tiles - 1 - w / per) * 256;
  t.len = diff_lens(p, t.b);
  const int last = min(t.r0 + 256, t.len.nq) - 1;
  t.kend = last >= t.r0 ? diff_limit(t.len, p.causal, last) : 0;
  t.nt = (t.kend + 127) / 128;
  t.ns = (t.kend + 63) / 64;
  return t;
}
// Whether step j of an item reaches behind its sequence's keys, so that the
// softmax warps clear rows of V: only the last step of a padded sequence.
__device__ __forceinline__ bool clears_v(const PairItem& t, const amc_diff_attention& p, int j) {
  return j * 64 + 64 > t.len.nk && t.len.nk < p.nk;
}

}  // namespace

template <typename T, int NV>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreadsF, 1)
    k_diff_fwd_pair(const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mK,
                    const __grid_constant__ CUtensorMap mV, const __grid_constant__ amc_diff_attention p) {
  using L = PairSmem;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char diff_sm_raw[];
  unsigned char* sm = (unsigned char*)(((uintptr_t)diff_sm_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* q_full = (uint64_t*)(sm + L::bar);    // this CTA's rows landed
  uint64_t* q_empty = q_full + 1;                 // the item's scores are complete
  uint64_t* kv_full = q_full + 2;                 // [kPStages] this CTA's halves landed
  uint64_t* kv_empty = kv_full + kPStages;        // [kPStages]
  uint64_t* s_full = kv_empty + kPStages;         // [buffer] both maps' scores complete
  uint64_t* acc_full = s_full + 2;                // the item's outputs complete
  // in the even CTA only:
  uint64_t* q_ready = acc_full + 1;               // both CTAs' rows landed (count 2)
  uint64_t* kv_ready = q_ready + 1;               // [kPStages] likewise
  uint64_t* p_full = kv_ready + kPStages;         // [buffer] P written (16 warps)
  uint64_t* o_free = p_full + 2;                  // the item's outputs are read (16 warps)
  uint32_t* tslot = (uint32_t*)(sm + L::bar + 240);
  volatile int* abort_flag = (volatile int*)(sm + L::bar + 244);
  const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int items = p.heads * p.batch * ((p.nq + 255) / 256), pairs = gridDim.x / 2, first = blockIdx.x / 2;
  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(q_ready, 2);
    for (int i = 0; i < kPStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
      mbar_init(&kv_ready[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 16);
    }
    mbar_init(acc_full, 1);
    mbar_init(o_free, 16);
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (warp == 0) tmem_alloc_pair(tslot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTA's barriers are set up
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tslot);   // S_m at 128 m + 64 (step & 1), O_m at 256 + 128 m

  if (warp == 8) {
    if (lane == 0) {
      int kt = 0, it = 0;   // tiles and (non-empty) items so far
      bool ok = true;
      for (int w = first; w < items && ok; w += pairs) {
        const PairItem t = pair_item(p, w);
        if (!t.ns) continue;
        if (it > 0) ok = mbar_wait(q_empty, (uint32_t)(it - 1) & 1u);
        if (!ok || *abort_flag) break;
        mbar_expect_tx(q_full, 32768);
        for (int m = 0; m < 2; ++m)
          tma_load_4d(sm + L::q + m * 16384, &mQ, 0, t.r0 + 128 * (int)rank, 2 * t.h + m, t.b, q_full);
        for (int j = 0; j < t.nt; ++j, ++kt) {
          const int s = kt % kPStages;
          if (kt >= kPStages) ok = mbar_wait(&kv_empty[s], (uint32_t)(kt / kPStages - 1) & 1u);
          if (!ok || *abort_flag) break;
          unsigned char* st = sm + L::kv + s * L::stage;
          mbar_expect_tx(&kv_full[s], L::stage);
          for (int c = 0; c < 2; ++c)
            for (int m = 0; m < 2; ++m)
              tma_load_4d(st + c * 8192 + m * 4096, &mK, 0, j * 128 + c * 64 + 32 * (int)rank, 2 * t.g + m, t.b,
                          &kv_full[s]);
          tma_load_4d(st + L::v, &mV, NV / 2 * (int)rank, j * 128, t.g, t.b, &kv_full[s]);
        }
        ++it;
      }
      // the last commits to this CTA's barriers have arrived before it may exit
      for (int i = max(0, kt - kPStages); i < kt && ok; ++i)
        ok = mbar_wait(&kv_empty[i % kPStages], (uint32_t)(i / kPStages) & 1u);
      if (ok && it > 0) ok = mbar_wait(q_empty, (uint32_t)(it - 1) & 1u);
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 10) {
    if (lane == 0) {
      int kt = 0, it = 0;
      bool ok = true;
      for (int w = first; w < items && ok; w += pairs) {
        const PairItem t = pair_item(p, w);
        if (!t.ns) continue;
        ok = mbar_wait(q_full, (uint32_t)it & 1u);
        if (ok) mbar_arrive_release_at(q_ready, 0);
        for (int j = 0; j < t.nt && ok; ++j, ++kt) {
          const int s = kt % kPStages;
          ok = mbar_wait(&kv_full[s], (uint32_t)(kt / kPStages) & 1u) && !*abort_flag;
          if (ok) mbar_arrive_release_at(&kv_ready[s], 0);
        }
        ++it;
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 9) {
    if (rank == 0) {
      const uint32_t id_s = idesc_f16(256, 64, kBf16, false, false);
      const uint32_t id_o = idesc_f16(256, NV, kBf16, false, true);
      const uint64_t qd = sdesc(smem_addr(sm + L::q), 16, 1024), kd = sdesc(smem_addr(sm + L::kv), 16, 1024);
      const uint64_t vd = sdesc_mn16(smem_addr(sm + L::kv + L::v), 16384);
      uint32_t slot = 0, lap = 0, it = 0;   // stage and phase of the item's first tile; items before it
      uint32_t step = 0;                    // steps before it (their parity is all that counts)
      bool ok = true;
      for (int w = first; w < items && ok; w += pairs) {
        const PairItem t = pair_item(p, w);
        const int ns = (int)warp_uniform(t.ns);
        if (!ns) continue;
        uint32_t ks = slot, kl = lap, vs = slot;   // K is used two steps ahead of V
        // scores of step j, both maps; j >= ns: the barrier alone
        auto issue_s = [&](int j) {
          const uint32_t buf = warp_uniform((step + j) & 1);
          if (j < ns) {
            // uniform by construction: all that an issue reads stays in uniform registers
            const uint64_t kb = desc_add(kd, warp_uniform(ks * L::stage + (j & 1) * 8192));
            const uint32_t d = tmem + buf * 64;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_f16_pair(d + m * 128, desc_add(qd, m * 16384 + k * 32), desc_add(kb, m * 4096 + k * 32), id_s, k > 0);
            if ((j & 1) && ++ks == kPStages) {
              ks = 0;
              kl ^= 1;
            }
          }
          mma_commit_pair(&s_full[buf]);
          if (j + 1 == ns) mma_commit_pair(q_empty);
        };
        ok = warp_wait_cluster(q_ready, it & 1) && warp_wait_cluster(&kv_ready[ks], kl);
        if (!ok) break;
        tc_fence_after();
        issue_s(0);
        issue_s(1);
        for (int j = 0; j < ns; ++j) {
          const uint32_t buf = warp_uniform((step + j) & 1);
          if (!(j & 1) && j + 2 < ns) ok = warp_wait_cluster(&kv_ready[ks], kl);
          if (ok && j == 0 && it > 0) ok = warp_wait(o_free, (it - 1) & 1);
          // where a step cleared rows of V, those stores have to reach the products of both CTAs
          ok = ok && (clears_v(t, p, j) ? warp_wait_cluster(&p_full[buf], ((step + j) >> 1) & 1)
                                        : warp_wait(&p_full[buf], ((step + j) >> 1) & 1));
          if (!ok) break;
          tc_fence_after();
          const uint64_t vb = desc_add(vd, warp_uniform(vs * L::stage + (j & 1) * 8192));
          const uint32_t pa = tmem + buf * 64;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_f16_pair_ts(tmem + 256 + m * 128, pa + m * 128 + k * 8, desc_add(vb, k * 2048), id_o, j > 0 || k > 0);
          issue_s(j + 2);
          if ((j & 1) || j + 1 == ns) {
            mma_commit_pair(&kv_empty[vs]);
            if (++vs == kPStages) {
              vs = 0;
              lap ^= 1;
            }
          }
        }
        if (ok) mma_commit_pair(acc_full);
        slot = vs;
        step += ns;
        ++it;
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    // ---------------- softmax of map m, one thread per query row
    const int m = warp >> 2, t = tid & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + m * 128 + lane_base, t_o = tmem + 256 + m * 128 + lane_base;
    const float c2 = p.scale * kLog2e;
    float* xch = (float*)(sm + L::x);
    int kt = 0, st = 0, it = 0;
    bool ok = true;
    for (int w = first; w < items && ok; w += pairs) {
      const PairItem a = pair_item(p, w);
      const int r0 = a.r0 + 128 * (int)rank, row = r0 + t;
      const int lim = diff_limit(a.len, p.causal, row);
      // steps that end at or below this need no mask in any row of the CTA
      const int all_see = r0 + 127 < a.len.nq ? diff_limit(a.len, p.causal, r0) : 0;
      float top = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
      for (int j = 0; j < a.ns; ++j) {
        // the barriers of scores count two more an item than its steps
        const int buf = (st + j) & 1, sj = st + 2 * it + j;
        const uint32_t t_b = t_s + buf * 64;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buf], (uint32_t)(sj >> 1) & 1u));
        if (!ok) break;
        tc_fence_after();
        uint32_t sr[2][32];
        tmem_ld32_nowait(t_b, sr[0]);
        tmem_ld32_nowait(t_b + 32, sr[1]);
        tmem_ld_wait();
        const bool masked = j * 64 + 64 > all_see, clears = clears_v(a, p, j);
        if (masked) {
          const int n = lim - j * 64;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * c + i >= n) sr[c][i] = 0xff800000u;
          if (clears) {
            // V behind the length may hold anything, and 0 times it is not 0:
            // clear those rows of this CTA's half before any product reads them
            const int i = kt + (j >> 1), r = (j & 1) * 64 + (t & 63);
            ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[i % kPStages], (uint32_t)(i / kPStages) & 1u));
            if (!ok) break;
            if ((j >> 1) * 128 + r >= a.len.nk) {
              unsigned char* vr = sm + L::kv + i % kPStages * L::stage + L::v + r * 128 + (t >> 6) * 64;
#pragma unroll
              for (int c = 0; c < 4; ++c) *reinterpret_cast<int4*>(vr + 16 * c) = make_int4(0, 0, 0, 0);
            }
            fence_proxy_async();
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
        const float mt = c2 * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool up = mt > top + 8.f;
        if (__any_sync(0xffffffffu, up)) {
          const float corr = up ? ex2_approx(top - mt) : 1.f;   // 0 at the first key
          if (up) {
            l2 = mul2(l2, make_float2(corr, corr));
            top = mt;
          }
          if (j > 0) {
            // P V of step j - 1 is complete when the scores of j + 1 are
            ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buf ^ 1], (uint32_t)((sj + 1) >> 1) & 1u));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < NV; c += 16) {
              float v[16];
              tmem_ld16(t_o + c, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] *= corr;
              tmem_st16(t_o + c, v);
            }
          }
        }
        const float base = top == -INFINITY ? 0.f : top;   // a row that has seen no key
        const float2 cc = make_float2(c2, c2), nb = make_float2(-base, -base);
        float2 s4[4] = {};
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 x = fma2(make_float2(__uint_as_float(sr[i >> 4][2 * (i & 15)]),
                                            __uint_as_float(sr[i >> 4][2 * (i & 15) + 1])), cc, nb);
          const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          s4[i & 3] = add2(s4[i & 3], e);
          v[i] = __uint_as_float(pack2<T>(e.x, e.y));
        }
        tmem_st32(t_b, v);
        tmem_st_wait();
        l2 = add2(l2, add2(add2(s4[0], s4[1]), add2(s4[2], s4[3])));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (clears) mbar_arrive_release_at(&p_full[buf], 0);
          else mbar_arrive_at(&p_full[buf], 0);
        }
      }
      if (a.ns > 0 && ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(acc_full, (uint32_t)it & 1u));
        tc_fence_after();
      }
      const float l = l2.x + l2.y;
      float f0 = 0.f, f1 = 0.f;
      if (a.ns > 0) {
        xch[m * 128 + t] = l != 0.f ? 1.f / l : 0.f;
        ok = named_bar_and(1, 256, ok && !*abort_flag);
        f0 = xch[t];
        f1 = xch[128 + t];
      }
      if (!ok) break;
      const float lam = lam_of<T>(p, a.h);
      if (p.lse && row < p.nq)
        p.lse[((int64_t)a.b * 2 * p.heads + 2 * a.h + m) * p.nq + row] = row_lse(top, l);
      // warpgroup m writes columns 64 m .. of both results (NV = 64: group 0 alone)
      if (64 * m < NV) {
        T* o = (T*)p.o + a.b * p.os[0] + a.h * p.os[1] + (int64_t)row * p.os[2] + 64 * m;
        T* o2 = p.o2 ? (T*)p.o2 + a.b * p.o2s[0] + a.h * p.o2s[1] + (int64_t)row * p.o2s[2] + 64 * m : nullptr;
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          float a0[16], a1[16];
          if (a.ns > 0) {
            tmem_ld16(tmem + 256 + lane_base + 64 * m + c, a0);
            tmem_ld16(tmem + 384 + lane_base + 64 * m + c, a1);
          }
          uint32_t w0[8], w2[8];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            a1[i] = a.ns > 0 ? a1[i] * f1 : 0.f;
            a0[i] = a.ns > 0 ? fmaf(-lam, a1[i], a0[i] * f0) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            w0[i] = pack2<T>(a0[2 * i], a0[2 * i + 1]);
            w2[i] = pack2<T>(a1[2 * i], a1[2 * i + 1]);
          }
          if (row < p.nq) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (64 * m + c + 8 * i < p.dv) {
                *reinterpret_cast<uint4*>(o + c + 8 * i) = make_uint4(w0[4 * i], w0[4 * i + 1], w0[4 * i + 2], w0[4 * i + 3]);
                if (o2)
                  *reinterpret_cast<uint4*>(o2 + c + 8 * i) = make_uint4(w2[4 * i], w2[4 * i + 1], w2[4 * i + 2], w2[4 * i + 3]);
              }
          }
        }
      }
      if (a.ns > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(o_free, 0);
        kt += a.nt;
        st += a.ns;
        ++it;
      }
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (tid == 0) atomicExch(&g_diff_error, AMC_ERR_TIMEOUT);
    // bounded drain of copies and products still in flight
    mbar_wait(q_full, 0, 1 << 14);
    for (int i = 0; i < kPStages; ++i) mbar_wait(&kv_full[i], 0, 1 << 14);
    for (int i = 0; i < 2; ++i) mbar_wait(&s_full[i], 0, 1 << 14);
    mbar_wait(acc_full, 0, 1 << 14);
    __syncthreads();
  }
  cluster_sync();   // the other CTA's products read this one's memory, and its warps arrive here
  if (warp == 0) tmem_dealloc_pair(tmem, 512);
}

namespace {

bool aligned_rows(const void* x, const int64_t s[3], const amc_diff_attention& p) {
  return !((uintptr_t)x & 15) && (p.batch == 1 || s[0] % 8 == 0) && (p.heads == 1 || s[1] % 8 == 0) &&
         (p.nq == 1 || s[2] % 8 == 0);
}

template <typename T, int NV>
int fwd_tc(const amc_diff_attention& p, const CUtensorMap (&map)[3], cudaStream_t s) {
  static std::atomic<uint64_t> attr{0};
  if (int rc = smem_attr_once(k_diff_fwd_tc<T, NV>, FwdSmem<NV>::bytes, attr)) return rc;
  const int64_t grid = (int64_t)((p.nq + 127) / 128) * p.heads * p.batch;
  k_diff_fwd_tc<T, NV><<<(unsigned)grid, kThreadsF, FwdSmem<NV>::bytes, s>>>(map[0], map[1], map[2], p);
  AMC_CUDA(cudaGetLastError());
  return AMC_OK;
}

template <typename T, int NV>
int fwd_pair(const amc_diff_attention& p, const CUtensorMap (&map)[3], cudaStream_t s) {
  static std::atomic<uint64_t> attr{0};
  if (int rc = smem_attr_once(k_diff_fwd_pair<T, NV>, PairSmem::bytes, attr)) return rc;
  const int64_t items = (int64_t)((p.nq + 255) / 256) * p.heads * p.batch;
  const int64_t pairs = items < num_sms() / 2 ? items : num_sms() / 2;
  k_diff_fwd_pair<T, NV><<<(unsigned)(2 * pairs), kThreadsF, PairSmem::bytes, s>>>(map[0], map[1], map[2], p);
  AMC_CUDA(cudaGetLastError());
  return AMC_OK;
}

}  // namespace

bool diff_tc_shape(const amc_diff_attention& p) {
  return p.dtype != AMC_F32 && p.d <= 64 && p.dv <= 128 && p.d % 8 == 0 && p.dv % 8 == 0 && p.nk > 0;
}

int diff_fwd_tc(const amc_diff_attention& p, cudaStream_t s, bool* handled) {
  *handled = false;
  // the running maximum is taken before the scale
  if (!diff_tc_shape(p) || !(p.scale > 0.f) || !aligned_rows(p.o, p.os, p) || (p.o2 && !aligned_rows(p.o2, p.o2s, p))) return AMC_OK;
  if ((int64_t)((p.nq + 127) / 128) * p.heads * p.batch > 0x7fffffff) return AMC_OK;
  CUtensorMap map[3];
  // Pairs halve what a row asks of the L2 and with it the power that limits long
  // runs, and load a tile behind the one before; but their step takes longer, a
  // causal mask leaves them uneven rounds, and a half-empty last tile costs two SMs.
  // In loops of calls, d 64, us on single CTAs against pairs: no mask, 1024 tiles
  // of 256 rows over 2048 keys 597 : 543, over 512 keys 207 : 181, 512 tiles over
  // 1024 150 : 144, 160 over 512 63 : 62; on the other side over 4096 keys 451 : 468,
  // over 16384 1495 : 1846, 777 rows and keys 174 : 187, causal 4096 x 4096 446 : 538,
  // 2048 x 2048 335 : 335, 777 x 777 129 : 154, and 80 to 128 tiles 65 : 72 and 68 : 73.
  const int64_t tiles = (int64_t)((p.nq + 255) / 256) * p.heads * p.batch;
  const bool bf16 = p.dtype == AMC_BF16;
  const bool pair = !p.causal && p.nk <= 2048 && (p.nq - 1) % 256 >= 128 && tiles >= 2 * (num_sms() / 2);
  int rc = make_tmap_4d_16(&map[0], p.q, bf16, p.batch, 2 * p.heads, p.nq, p.d, p.qs, 128);
  if (!rc) rc = make_tmap_4d_16(&map[1], p.k, bf16, p.batch, 2 * p.kv_heads, p.nk, p.d, p.ks, pair ? 32 : 128);
  if (!rc) rc = make_tmap_4d_16(&map[2], p.v, bf16, p.batch, p.kv_heads, p.nk, p.dv, p.vs, 128);
  if (rc == AMC_ERR_UNSUPPORTED) return AMC_OK;
  if (rc) return rc;
  *handled = true;
  if (pair && bf16) return p.dv <= 64 ? fwd_pair<__nv_bfloat16, 64>(p, map, s) : fwd_pair<__nv_bfloat16, 128>(p, map, s);
  if (pair) return p.dv <= 64 ? fwd_pair<__half, 64>(p, map, s) : fwd_pair<__half, 128>(p, map, s);
  if (bf16) return p.dv <= 64 ? fwd_tc<__nv_bfloat16, 64>(p, map, s) : fwd_tc<__nv_bfloat16, 128>(p, map, s);
  return p.dv <= 64 ? fwd_tc<__half, 64>(p, map, s) : fwd_tc<__half, 128>(p, map, s);
}

int diff_check_error() {
  int e = 0;
  AMC_CUDA(cudaMemcpyFromSymbol(&e, g_diff_error, sizeof(int)));
  if (e) {
    int z = 0;
    AMC_CUDA(cudaMemcpyToSymbol(g_diff_error, &z, sizeof(int)));
    return fail(e, "diff_attention: a bounded wait on the tensor-core pipeline gave up");
  }
  return AMC_OK;
}

}  // namespace amc
