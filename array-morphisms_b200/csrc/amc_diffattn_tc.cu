// Differential attention forward on the tensor cores (sm_100a, tcgen05
// kind::f16), 16-bit tensors with d <= 64 and dv <= 128, both multiples of 8.
//
// A CTA owns 128 query rows of one head.  Its two maps are two warpgroups,
// one thread per row, that share the V tile; 128-key tiles stream through
// shared memory by TMA (smaller heads are zero-filled to 64 / NV columns).
// Warp 8 loads, warp 9 issues, in the order
//   S0(0) S1(0) | PV0(0) S0(1) PV1(0) S1(1) | PV0(1) ...
// so that one map's products run while the other map is in its softmax.
// Tensor memory holds S_0, S_1 (128 columns each) and O_0, O_1 (NV each):
// all 512 columns at NV = 128, which is why one CTA takes exactly one tile of
// both maps.  P goes back over its own S as 16-bit pairs and is the A operand
// of P V from there; V is an MN-major operand, read as TMA wrote it.
//   p = 2^(scale log2e s - m), rounded to the tensors' type for P V and
//   summed unrounded; m follows the row maximum only when it rises by more
//   than 2^8, and O is rescaled then, once the group's earlier products are
//   complete (the completion of S(j) implies that of PV(j-1), issued before).
// The two rows' results meet in the epilogue: O = O_0 / l_0 - lam O_1 / l_1.
//
// Bound: per 128 x 128 tile of both maps the products take 1536 clocks of the
// tensor pipe and the 32768 exponentials 2048 of the special-function unit.
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

constexpr int kThreadsF = 320;
constexpr int kKStages = 3, kVStages = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994530942f;

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

// lam of head h on every lane (the warp is converged).
template <typename T>
__device__ __forceinline__ float lam_of(const amc_diff_attention& p, int h) {
  const T* l = (const T*)p.lam + (size_t)(p.lam_rows == 1 ? 0 : h) * 4 * p.d;
  float a = 0.f, c = 0.f;
  for (int i = threadIdx.x & 31; i < p.d; i += 32) {
    a = fmaf(to_f32(l[i]), to_f32(l[p.d + i]), a);
    c = fmaf(to_f32(l[2 * p.d + i]), to_f32(l[3 * p.d + i]), c);
  }
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  return expf(a) - expf(c) + p.lam_init;
}

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
  uint64_t* s_full = v_empty + kVStages;          // [2] per map: S(j) (and PV(j-1)) complete
  uint64_t* p_full = s_full + 2;                  // [2] per map: P(j) written (count 128)
  uint64_t* o_done = p_full + 2;
  uint32_t* tslot = (uint32_t*)(sm + L::bar + 192);
  volatile int* abort_flag = (volatile int*)(sm + L::bar + 196);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // Tiles of one head are launched last row tile first (with a causal mask
  // those see the most keys), the heads of one key head next to each other.
  const int per = p.heads * p.batch, tiles = (p.nq + 127) / 128;
  const int tile = tiles - 1 - (int)(blockIdx.x / per), h = blockIdx.x % per % p.heads, b = blockIdx.x % per / p.heads;
  const int g = h / (p.heads / p.kv_heads), r0 = tile * 128;
  const DiffLens len = diff_lens(p, b);
  const int last = min(r0 + 128, len.nq) - 1;
  const int kend = last >= r0 ? diff_limit(len, p.causal, last) : 0;
  const int nt = (kend + 127) / 128;
  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kKStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    mbar_init(o_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (warp == 0) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;   // S_g at 128 g, O_g at 256 + 128 g

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
  } else if (warp == 9) {
    if (lane == 0 && nt > 0) {
      const uint32_t id_s = idesc_f16(128, 128, kBf16, false, false);
      const uint32_t id_o = idesc_f16(128, NV, kBf16, false, true);
      const uint64_t qd = sdesc(smem_addr(sm + L::q), 16, 1024), kd = sdesc(smem_addr(sm + L::k), 16, 1024);
      const uint64_t vd = sdesc_mn16(smem_addr(sm + L::v), 16384);
      const int ksteps = (p.d + 15) / 16;
      auto issue_s = [&](int m, int j) {
        const uint64_t qb = desc_add(qd, m * 16384), kb = desc_add(kd, (j % kKStages) * 32768 + m * 16384);
        for (int k = 0; k < ksteps; ++k)
          mma_f16(tmem + m * 128, desc_add(qb, k * 32), desc_add(kb, k * 32), id_s, k > 0);
        mma_commit(&s_full[m]);
      };
      auto issue_pv = [&](int m, int j) {
        const uint64_t vb = desc_add(vd, (j % kVStages) * L::v_bytes);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_f16_ts(tmem + 256 + m * 128, tmem + m * 128 + k * 8, desc_add(vb, k * 2048), id_o, j > 0 || k > 0);
      };
      bool ok = mbar_wait(q_full, 0) && mbar_wait(&k_full[0], 0);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        issue_s(1, 0);
        mma_commit(&k_empty[0]);
      }
      for (int j = 0; j < nt && ok; ++j) {
        const int t = j % kVStages, s1 = (j + 1) % kKStages;
        const bool more = j + 1 < nt;
        if (!mbar_wait(&v_full[t], (uint32_t)(j / kVStages) & 1u)) { ok = false; break; }
        if (more && !mbar_wait(&k_full[s1], (uint32_t)((j + 1) / kKStages) & 1u)) { ok = false; break; }
        for (int m = 0; m < 2 && ok; ++m) {
          if (!mbar_wait(&p_full[m], (uint32_t)j & 1u) || *abort_flag) { ok = false; break; }
          tc_fence_after();
          issue_pv(m, j);
          if (m == 1) mma_commit(&v_empty[t]);
          if (more) issue_s(m, j + 1);
        }
        if (ok && more) mma_commit(&k_empty[s1]);
      }
      if (ok) mma_commit(o_done);
      else *abort_flag = 1;
    }
  } else {
    // ---------------- softmax of map m, one thread per query row
    const int m = warp >> 2, t = tid & 127, row = r0 + t;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + m * 128 + lane_base;
    const float c2 = p.scale * kLog2e;
    const int lim = diff_limit(len, p.causal, row);
    // tiles that end at or below this need no mask in any row of the CTA
    const int all_see = r0 + 127 < len.nq ? diff_limit(len, p.causal, r0) : 0;
    float top = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[m], (uint32_t)j & 1u) && !*abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32_nowait(t_s + 32 * c, sr[c]);
      tmem_ld_wait();
      if (j * 128 + 128 > all_see) {
        const int n = lim - j * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (32 * c + i >= n) sr[c][i] = 0xff800000u;
        if (j * 128 + 128 > len.nk && len.nk < p.nk) {
          // V behind the length may hold anything, and 0 times it is not 0:
          // clear those rows of the tile before any product reads it
          const int vs = j % kVStages;
          ok = __all_sync(0xffffffffu, mbar_wait(&v_full[vs], (uint32_t)(j / kVStages) & 1u));
          if (!ok) break;
          if (j * 128 + t >= len.nk) {
            unsigned char* vr = sm + L::v + vs * L::v_bytes + t * 128;
#pragma unroll
            for (int c = 0; c < NV / 64; ++c)
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<int4*>(vr + c * 16384 + 16 * i) = make_int4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
      }
      float mx8[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) mx8[k] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) mx8[i & 7] = fmaxf(mx8[i & 7], __uint_as_float(sr[c][i]));
      const float mt = c2 * fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                                  fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
      const bool up = mt > top + 8.f;
      if (__any_sync(0xffffffffu, up)) {
        const float corr = up ? ex2_approx(top - mt) : 1.f;   // 0 at the first key
        if (up) {
          l *= corr;
          top = mt;
        }
        if (j > 0) {
          const uint32_t t_o = tmem + 256 + m * 128 + lane_base;
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
      float sm8[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) sm8[k] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float p0 = ex2_approx(fmaf(__uint_as_float(sr[2 * c + (i >> 4)][2 * (i & 15)]), c2, -base));
          const float p1 = ex2_approx(fmaf(__uint_as_float(sr[2 * c + (i >> 4)][2 * (i & 15) + 1]), c2, -base));
          sm8[2 * i & 7] += p0;
          sm8[(2 * i + 1) & 7] += p1;
          v[i] = __uint_as_float(pack2<T>(p0, p1));
        }
        tmem_st32(t_s + 32 * c, v);
      }
      tmem_st_wait();
      l += ((sm8[0] + sm8[1]) + (sm8[2] + sm8[3])) + ((sm8[4] + sm8[5]) + (sm8[6] + sm8[7]));
      tc_fence_before();
      mbar_arrive(&p_full[m]);
    }
    if (nt > 0) ok = ok && mbar_wait(o_done, 0);
    const float lam = lam_of<T>(p, h);
    float* xch = (float*)(sm + L::x);
    xch[m * 128 + t] = l > 0.f ? 1.f / l : 0.f;
    ok = named_bar_and(1, 256, ok && !*abort_flag);
    if (ok) {
      // warpgroup m writes columns 64 m .. of both results (NV = 64: group 0 alone)
      tc_fence_after();
      if (row < p.nq) {
        if (p.lse) p.lse[((int64_t)b * 2 * p.heads + 2 * h + m) * p.nq + row] =
            l > 0.f ? fmaf(top, kLn2, logf(l)) : -INFINITY;
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
            a1[i] = nt > 0 ? a1[i] * f1 : 0.f;
            a0[i] = nt > 0 ? fmaf(f, a1[i], a0[i] * f0) : 0.f;
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
    for (int i = 0; i < 2; ++i) mbar_wait(&s_full[i], 0, 1 << 14);
    mbar_wait(o_done, 0, 1 << 14);
  }
  if (warp == 0) tmem_dealloc(tmem, 512);
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
  const bool bf16 = p.dtype == AMC_BF16;
  int rc = make_tmap_4d_16(&map[0], p.q, bf16, p.batch, 2 * p.heads, p.nq, p.d, p.qs, 128);
  if (!rc) rc = make_tmap_4d_16(&map[1], p.k, bf16, p.batch, 2 * p.kv_heads, p.nk, p.d, p.ks, 128);
  if (!rc) rc = make_tmap_4d_16(&map[2], p.v, bf16, p.batch, p.kv_heads, p.nk, p.dv, p.vs, 128);
  if (rc == AMC_ERR_UNSUPPORTED) return AMC_OK;
  if (rc) return rc;
  *handled = true;
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
