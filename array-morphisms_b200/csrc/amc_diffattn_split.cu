// Differential attention of few rows over many keys (the single-token form),
// 16-bit tensors with d <= 64 and dv <= 128, both multiples of 8.
//
// The bound is HBM: every key and value is read once, for all rows of its key
// head (the query heads that share it times their rows, 16 at most).  The keys of
// all sequences and key heads, in blocks of 64, are one line of work that the
// CTAs, two a SM, share evenly, so sequences of different lengths leave none
// idle; a CTA's share may end one sequence and begin another.
// Within a CTA the four warps take a block's four boxes of 16 keys.  Warps do
// not wait for each other: each has its own ring of TMA boxes (K_1, K_2 and V
// rows of 16 keys, 8 KB), its own running maximum, sum and output, and they
// meet at the end of a sequence's part in shared memory.  The products are
// mma.sync m16n8k16: 16 rows fill a legacy tile, where a tcgen05 tile of 128
// would be an eighth full, and at 16 rows they take less than half the time
// of the loads.  P is taken into P V as the sum of two 16-bit values (the
// rounded one and the rounding's remainder): the result carries no rounding of
// P.  With 8 rows or fewer the two maps share a tile of P, map 1 in its lower
// half, which takes 48 products a box instead of 80.  A second kernel joins the
// parts of the sequences that several CTAs worked on by their maxima and sums.
// Measured, 16 query heads (d 64, dv 128) over 4 key heads, 8 caches of up to
// 32768 keys (302 MB): 61 us without the join (4.9 TB/s) with the shared tile,
// 66 us with two; full caches (537 MB): 94 us, 5.7 TB/s.
#include <cmath>
#include <type_traits>

#include "amc_diffattn.h"
#include "amc_half.cuh"
#include "amc_tc.cuh"

namespace amc {

using namespace tc;

namespace {

constexpr int kRows = 16;            // rows per CTA
constexpr int kWarps = 4;
constexpr int kStages = 3;           // boxes in flight per warp
constexpr int kBox = 8192;           // 16 keys: K_1 2 KB, K_2 2 KB, V 4 KB
constexpr int kStageBytes = kWarps * kStages * kBox;
constexpr int kSplitSmem = kStageBytes + 512 + 1024;
constexpr int kShareCtas = 148 * 2;  // CTAs that share the keys: two a SM of the B200, and the workspace's size
constexpr int kMinShare = 4;         // blocks of 64 keys: 4 boxes a warp
constexpr int kMaxBatch = 1024;      // sequences whose lengths a CTA sums up
constexpr float kLog2e = 1.4426950408889634f;

__device__ int g_diff_split_error;

struct SplitArgs {
  int group, shared;   // shared: the keys are shared out (else a unit a CTA)
  float* part;       // [CTA][first or last unit][row][map][dv] unscaled outputs
  float2* part_ml;   // [CTA][first or last unit][row][map] maximum (log2 units) and sum
};

// A unit is one sequence and key head with its rows, 16 at most.  Its blocks of 64
// keys stand on one line after those of the units before it.
struct Unit {
  int b, g, blocks;      // sequence, key head, blocks
  int64_t first;         // its first block on the line
};
__device__ __forceinline__ int seq_blocks(const amc_diff_attention& p, int b) {
  const DiffLens len = diff_lens(p, b);
  return len.nq > 0 ? (len.nk + 63) / 64 : 0;
}
// All blocks of the line, by one warp.
__device__ __forceinline__ int64_t line_blocks(const amc_diff_attention& p, int per_seq) {
  int64_t n = 0;
  for (int b = threadIdx.x & 31; b < p.batch; b += 32) n += seq_blocks(p, b);
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * per_seq;
}
// The unit of block x, by one warp.
__device__ __forceinline__ Unit find_unit(const amc_diff_attention& p, int per_seq, int64_t x) {
  int64_t before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + (threadIdx.x & 31);
    const int64_t mine = b < p.batch ? (int64_t)seq_blocks(p, b) * per_seq : 0;
    int64_t upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if ((threadIdx.x & 31) >= o) upto += v;
    }
    const unsigned here = __ballot_sync(0xffffffffu, before + upto > x);
    if (here) {
      const int l = __ffs(here) - 1;
      Unit r;
      r.b = b0 + l;
      r.blocks = (int)(__shfl_sync(0xffffffffu, mine, l) / per_seq);
      const int64_t start = before + __shfl_sync(0xffffffffu, upto, l) - (int64_t)r.blocks * per_seq;
      r.g = (int)((x - start) / r.blocks);
      r.first = start + (int64_t)r.g * r.blocks;
      return r;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return Unit{0, 0, 0, x};
}
__device__ __forceinline__ int64_t share_of(int64_t total) {
  const int64_t n = (total + kShareCtas - 1) / kShareCtas;
  return n < kMinShare ? kMinShare : n;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// D (16 x 8, f32) += A (16 x 16) B (16 x 8)
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Row rr of a unit is query head g * group + rr / nq, row rr % nq.
__device__ __forceinline__ void unit_row(const amc_diff_attention& p, const SplitArgs& a, int g, int rr, int& h, int& i) {
  h = g * a.group + rr / p.nq;
  i = rr % p.nq;
}

template <typename T>
__device__ __forceinline__ void put_result(const amc_diff_attention& p, int b, int h, int i, int c, float o0, float o1) {
  ((T*)p.o)[b * p.os[0] + h * p.os[1] + (int64_t)i * p.os[2] + c] = from_f32<T>(o0);
  if (p.o2) ((T*)p.o2)[b * p.o2s[0] + h * p.o2s[1] + (int64_t)i * p.o2s[2] + c] = from_f32<T>(o1);
}

}  // namespace

template <typename T, int NV, bool PACK>
__global__ void __launch_bounds__(kWarps * 32) k_diff_split(const __grid_constant__ CUtensorMap mK,
                                                           const __grid_constant__ CUtensorMap mV,
                                                           const __grid_constant__ amc_diff_attention p,
                                                           const __grid_constant__ SplitArgs a) {
  constexpr int NT = NV / 8, RR = PACK ? 1 : 2;   // rows of a lane and map
  extern __shared__ unsigned char diff_sm_raw[];
  unsigned char* sm = (unsigned char*)(((uintptr_t)diff_sm_raw + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, pos = lane & 3;
  uint64_t* full = (uint64_t*)(sm + kStageBytes) + warp * kStages;
  volatile int* failed = (volatile int*)(sm + kStageBytes + 256);
  const int per_seq = p.kv_heads;
  int64_t at, end;   // this CTA's blocks on the line
  Unit first_unit{0, 0, 0, 0};
  if (a.shared) {
    const int64_t total = line_blocks(p, per_seq), share = share_of(total);
    at = share * blockIdx.x;
    end = at + share < total ? at + share : total;
    if (at >= end) {
      if (blockIdx.x) return;
      end = at;
    }
  } else {
    first_unit.b = blockIdx.x / per_seq;
    first_unit.g = blockIdx.x % per_seq;
    first_unit.blocks = seq_blocks(p, first_unit.b);
    at = 0;
    end = first_unit.blocks;
  }
  asm volatile("griddepcontrol.launch_dependents;");
  unsigned char* ring = sm + warp * kStages * kBox;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    if (warp == 0) *failed = 0;
    mbar_fence_init();
  }
  __syncthreads();
  const int64_t begin = at;
  int used = 0;   // boxes of this warp before this part
  do {
  const Unit unit = a.shared ? find_unit(p, per_seq, at) : first_unit;
  const int g = unit.g, b = unit.b, rows = a.group * p.nq;
  const DiffLens len = diff_lens(p, b);
  const int64_t stop = min(end, unit.first + unit.blocks);
  const int kbeg = (int)(at - unit.first) * 64, kend = min(len.nq > 0 ? len.nk : 0, (int)(stop - unit.first) * 64);
  int lim[RR];    // keys that this lane's rows see
#pragma unroll
  for (int r = 0; r < RR; ++r) {
    const int rr = quad + 8 * r;
    int h, i;
    unit_row(p, a, g, min(rr, rows - 1), h, i);
    lim[r] = rr < rows ? diff_limit(len, p.causal, i) : 0;
  }
  // box n of this warp starts at key kbeg + 16 (warp + 4 n)
  const int boxes = kend > kbeg ? (kend - kbeg + 15) / 16 : 0;
  const int mine = boxes > warp ? (boxes - warp + kWarps - 1) / kWarps : 0;
  auto load = [&](int n) {
    const int s = (used + n) % kStages;
    unsigned char* st = ring + s * kBox;
    const int key = kbeg + 16 * (warp + kWarps * n);
    mbar_expect_tx(&full[s], 4096 + NV / 64 * 2048);
    tma_load_4d(st, &mK, 0, key, 2 * g, b, &full[s]);
    tma_load_4d(st + 2048, &mK, 0, key, 2 * g + 1, b, &full[s]);
    for (int c = 0; c < NV / 64; ++c) tma_load_4d(st + 4096 + c * 2048, &mV, 64 * c, key, g, b, &full[s]);
  };
  if (lane == 0)
    for (int n = 0; n < kStages && n < mine; ++n) load(n);
  // Q fragments: rows quad and quad + 8, columns 16 k + 2 pos (+8)
  uint32_t q[2][4][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (r >= RR) {
#pragma unroll
        for (int k = 0; k < 4; ++k) q[m][k][r] = q[m][k][r + 2] = 0u;
        continue;
      }
      int h, i;
      unit_row(p, a, g, min(quad + 8 * r, rows - 1), h, i);
      const T* src = (const T*)p.q + b * p.qs[0] + (2 * h + m) * p.qs[1] + (int64_t)i * p.qs[2];
      const bool use = quad + 8 * r < rows && i < len.nq;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 16 * k + 8 * e + 2 * pos;
          q[m][k][r + 2 * e] = use && c < p.d ? *reinterpret_cast<const uint32_t*>(src + c) : 0u;
        }
    }
  const float c2 = p.scale * kLog2e;
  float top[2][RR], sum[2][RR], o[RR][NT][4];   // PACK: one output, map m in registers 2 m, 2 m + 1
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      top[m][r] = -INFINITY;
      sum[m][r] = 0.f;
    }
#pragma unroll
  for (int m = 0; m < RR; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
  const int mrow = lane & 7, mid = lane >> 3;   // ldmatrix: row and matrix of this lane's address
  bool ok = true;
  for (int n = 0; n < mine; ++n) {
    const int s = (used + n) % kStages;
    unsigned char* st = ring + s * kBox;
    const int key = kbeg + 16 * (warp + kWarps * n);
    ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (uint32_t)((used + n) / kStages) & 1u));
    if (!ok) break;
    if (key + 16 > len.nk && len.nk < p.nk) {
      // V behind the length may hold anything, and 0 times it is not 0
      const int r = lane & 15;
      if (key + r >= len.nk && (lane >> 4) < NV / 64)
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<int4*>(st + 4096 + (lane >> 4) * 2048 + r * 128 + 16 * c) = make_int4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
    }
    uint32_t ph[RR][4], pl[RR][4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float sc[2][4] = {};
      const uint32_t kb = smem_addr(st + m * 2048) + (mrow + (mid >> 1) * 8) * 128;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t f[4];
        ldsm4(f, kb + (((2 * k + (mid & 1)) ^ mrow) << 4));
        mma16<T>(sc[0], q[m][k], f[0], f[1]);
        mma16<T>(sc[1], q[m][k], f[2], f[3]);
      }
      if (key + 16 > min(lim[0], lim[RR - 1])) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2 * RR; ++e)
            if (key + 8 * t + 2 * pos + (e & 1) >= lim[e >> 1]) sc[t][e] = -INFINITY;
      }
      bool up = false;
      float mt[RR];
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        float x = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        mt[r] = x * c2;
        up = up || mt[r] > top[m][r] + 8.f;
      }
      if (__any_sync(0xffffffffu, up)) {
        // raise the maxima that lag by more than 2^8
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          const bool raise = mt[r] > top[m][r] + 8.f;
          const float corr = raise ? ex2_approx(top[m][r] - mt[r]) : 1.f;
          if (raise) top[m][r] = mt[r];
          sum[m][r] *= corr;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            o[PACK ? 0 : m][t][2 * (PACK ? m : r)] *= corr;
            o[PACK ? 0 : m][t][2 * (PACK ? m : r) + 1] *= corr;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          const float base = top[m][r] == -INFINITY ? 0.f : top[m][r];
          const float p0 = ex2_approx(fmaf(sc[t][2 * r], c2, -base)), p1 = ex2_approx(fmaf(sc[t][2 * r + 1], c2, -base));
          sum[m][r] += p0 + p1;
          const uint32_t hi = pack2<T>(p0, p1);
          const float2 back = unpack2<T>(hi);
          ph[PACK ? 0 : m][2 * t + (PACK ? m : r)] = hi;
          pl[PACK ? 0 : m][2 * t + (PACK ? m : r)] = pack2<T>(p0 - back.x, p1 - back.y);
        }
    }
#pragma unroll
    for (int t = 0; t < NT / 2; ++t) {
      uint32_t f[4];
      const int chunk = 2 * (t & 3) + (mid >> 1);
      ldsm4_t(f, smem_addr(st + 4096 + (t >> 2) * 2048) + (mrow + (mid & 1) * 8) * 128 + ((chunk ^ mrow) << 4));
#pragma unroll
      for (int m = 0; m < RR; ++m) {
        mma16<T>(o[m][2 * t], ph[m], f[0], f[1]);
        mma16<T>(o[m][2 * t + 1], ph[m], f[2], f[3]);
        mma16<T>(o[m][2 * t], pl[m], f[0], f[1]);
        mma16<T>(o[m][2 * t + 1], pl[m], f[2], f[3]);
      }
    }
    __syncwarp();
    if (lane == 0 && n + kStages < mine) load(n + kStages);
  }
  if (!ok) {
    if (lane == 0) {
      *failed = 1;
      atomicExch(&g_diff_split_error, AMC_ERR_TIMEOUT);
      for (int s = 0; s < kStages; ++s) mbar_wait(&full[s], 0, 1 << 14);
    }
  }
  // ---- join the four warps: rows' maxima, then sums and outputs over them
  __syncthreads();
  if (*failed) return;
  float* xo = (float*)sm;                                   // [warp][map][row][NV]
  float2* xml = (float2*)(sm + kWarps * 2 * kRows * NV * 4); // [warp][map][row]
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      float l = sum[m][r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int row = quad + 8 * r;
      if (pos == 0) xml[(warp * 2 + m) * kRows + row] = make_float2(top[m][r], l);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<float2*>(xo + ((warp * 2 + m) * kRows + row) * NV + 8 * t + 2 * pos) =
            make_float2(o[PACK ? 0 : m][t][2 * (PACK ? m : r)], o[PACK ? 0 : m][t][2 * (PACK ? m : r) + 1]);
    }
  __syncthreads();
  for (int row = warp; row < rows; row += kWarps) {
    int h, i;
    unit_row(p, a, g, row, h, i);
    float mx[2], l[2], acc[2][NV / 32];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      mx[m] = -INFINITY;
      for (int w = 0; w < kWarps; ++w) mx[m] = fmaxf(mx[m], xml[(w * 2 + m) * kRows + row].x);
      const float base = mx[m] == -INFINITY ? 0.f : mx[m];
      l[m] = 0.f;
#pragma unroll
      for (int c = 0; c < NV / 32; ++c) acc[m][c] = 0.f;
      for (int w = 0; w < kWarps; ++w) {
        const float2 e = xml[(w * 2 + m) * kRows + row];
        const float f = exp2f(e.x - base);
        l[m] = fmaf(e.y, f, l[m]);
#pragma unroll
        for (int c = 0; c < NV / 32; ++c)
          acc[m][c] = fmaf(xo[((w * 2 + m) * kRows + row) * NV + 32 * c + lane], f, acc[m][c]);
      }
    }
    if (a.shared && stop - at < unit.blocks) {
      // part of a unit: the end of one that this CTA's share begins with, or
      // (or also) the beginning of one
      const int64_t slot = (((int64_t)blockIdx.x * 2 + (at > begin)) * kRows + row) * 2;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (lane == 0) a.part_ml[slot + m] = make_float2(mx[m], l[m]);
#pragma unroll
        for (int c = 0; c < NV / 32; ++c)
          if (32 * c + lane < p.dv) a.part[(slot + m) * p.dv + 32 * c + lane] = acc[m][c];
      }
    } else {
      const float lam = lam_of<T>(p, h);
      const float f0 = l[0] != 0.f ? 1.f / l[0] : 0.f, f1 = l[1] != 0.f ? 1.f / l[1] : 0.f;
#pragma unroll
      for (int c = 0; c < NV / 32; ++c) {
        const float o1 = acc[1][c] * f1;
        if (32 * c + lane < p.dv) put_result<T>(p, b, h, i, 32 * c + lane, fmaf(-lam, o1, acc[0][c] * f0), o1);
      }
      if (p.lse && lane < 2) {
        const float ll = lane ? l[1] : l[0], mm = lane ? mx[1] : mx[0];
        p.lse[((int64_t)b * 2 * p.heads + 2 * h + lane) * p.nq + i] = row_lse(mm, ll);
      }
    }
  }
  used += mine;
  at = stop;
  __syncthreads();   // the exchange is read before the next part's boxes land there
  fence_proxy_async();
  } while (at < end);
}

// One CTA per (batch, head, row) of the sequences that several CTAs worked on,
// and of those without a key: the parts' outputs over their joint maxima.
template <typename T>
__global__ void __launch_bounds__(256) k_diff_join(const __grid_constant__ amc_diff_attention p,
                                                   const __grid_constant__ SplitArgs a) {
  __shared__ float2 ml[2][kShareCtas + 1];
  __shared__ float other[256];
  const int i = blockIdx.x % p.nq, h = blockIdx.x / p.nq % p.heads, b = blockIdx.x / p.nq / p.heads;
  const int g = h / a.group, rr = (h - g * a.group) * p.nq + i, per_seq = p.kv_heads;
  const int tid = threadIdx.x, m = tid >> 7, c = tid & 127;
  const int blocks = seq_blocks(p, b);
  int n = 0, c0 = 0;
  int64_t first = 0, share = 1;
  if (blocks) {
    // this unit's place on the line: the blocks of the sequences before, by every warp
    int64_t before = 0, total = 0;
    for (int q = tid & 31; q < p.batch; q += 32) {
      const int64_t s = seq_blocks(p, q);
      total += s;
      if (q < b) before += s;
    }
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    share = share_of(total * per_seq);
    first = before * per_seq + (int64_t)g * blocks;
    c0 = (int)(first / share);
    n = (int)((first + blocks - 1) / share) - c0 + 1;
  }
  // The first kernel lets this one start early: its results (and the launch after
  // this one, which must not pass it) wait for it here, every thread of the grid.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n == 1) return;   // one CTA saw all its keys and wrote the result
  // CTA c0 + k holds this unit as its first, but for c0 itself if its share began before
  auto slot = [&](int k) -> int64_t {
    const int second = k == 0 && first > c0 * share;
    return (((int64_t)(c0 + k) * 2 + second) * kRows + rr) * 2 + m;
  };
  for (int k = c; k < n; k += 128) ml[m][k] = a.part_ml[slot(k)];
  __syncthreads();
  float mx = -INFINITY, l = 0.f;
  for (int k = tid & 31; k < n; k += 32) mx = fmaxf(mx, ml[m][k].x);
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float base = mx == -INFINITY ? 0.f : mx;
  for (int k = tid & 31; k < n; k += 32) l = fmaf(ml[m][k].y, exp2f(ml[m][k].x - base), l);
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const float lam = lam_of<T>(p, h);
  for (int c1 = 0; c1 < p.dv; c1 += 128) {
    const int col = c1 + c;
    float acc = 0.f;
    if (col < p.dv) {
#pragma unroll 8
      for (int k = 0; k < n; ++k) acc = fmaf(a.part[slot(k) * p.dv + col], exp2f(ml[m][k].x - base), acc);
    }
    acc *= inv;
    other[tid] = acc;
    __syncthreads();
    if (m == 0 && col < p.dv) put_result<T>(p, b, h, i, col, fmaf(-lam, other[tid + 128], acc), other[tid + 128]);
    __syncthreads();
  }
  if (p.lse && c == 0)
    p.lse[((int64_t)b * 2 * p.heads + 2 * h + m) * p.nq + i] = row_lse(mx, l);
}

namespace {

SplitArgs plan(const amc_diff_attention& p) {
  SplitArgs a{};
  a.group = p.heads / p.kv_heads;
  // Units go to a CTA each where there are plenty of them, or where a cache
  // is so short that a second kernel would cost more than it shares out.
  const int64_t units = (int64_t)p.batch * p.kv_heads;
  a.shared = units < 2 * kShareCtas && p.batch <= kMaxBatch && p.nk > 64 * kMinShare;
  return a;
}

constexpr size_t kPartRows = (size_t)kShareCtas * 2 * kRows * 2;

template <typename T, int NV, bool PACK>
int split_main(const amc_diff_attention& p, const SplitArgs& a, const CUtensorMap (&map)[2], cudaStream_t s) {
  static std::atomic<uint64_t> attr{0};
  if (int rc = smem_attr_once(k_diff_split<T, NV, PACK>, kSplitSmem, attr)) return rc;
  const unsigned grid = a.shared ? kShareCtas : (unsigned)((int64_t)p.batch * p.kv_heads);
  k_diff_split<T, NV, PACK><<<grid, kWarps * 32, kSplitSmem, s>>>(map[0], map[1], p, a);
  AMC_CUDA(cudaGetLastError());
  return AMC_OK;
}

template <typename T, int NV>
int split_launch(const amc_diff_attention& p, const SplitArgs& a, const CUtensorMap (&map)[2], cudaStream_t s) {
  const bool pack = a.group * p.nq <= 8;
  if (int rc = pack ? split_main<T, NV, true>(p, a, map, s) : split_main<T, NV, false>(p, a, map, s)) return rc;
  if (a.shared) {
    // launched while the first kernel runs: 3 us less for both (75 to 72 us)
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((int64_t)p.batch * p.heads * p.nq));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    AMC_CUDA(cudaLaunchKernelEx(&cfg, k_diff_join<T>, p, a));
  }
  return AMC_OK;
}

}  // namespace

// The rows that share a key head fill at most one block: beyond that the
// 128-row kernel reads the keys fewer times.
static bool split_shape(const amc_diff_attention& p) {
  return diff_tc_shape(p) && p.nq > 0 && p.batch > 0 && (int64_t)(p.heads / p.kv_heads) * p.nq <= kRows;
}

size_t diff_split_bytes(const amc_diff_attention& p) {
  if (!split_shape(p) || !plan(p).shared) return 0;
  return kPartRows * (p.dv * sizeof(float) + sizeof(float2));
}

int diff_fwd_split(const amc_diff_attention& p, cudaStream_t s, bool* handled) {
  *handled = false;
  if (!split_shape(p) || !(p.scale > 0.f)) return AMC_OK;   // the running maximum is taken before the scale
  // Q is read in pairs
  if (((uintptr_t)p.q & 3) || (p.batch > 1 && p.qs[0] % 2) || p.qs[1] % 2 || (p.nq > 1 && p.qs[2] % 2)) return AMC_OK;
  CUtensorMap map[2];
  const bool bf16 = p.dtype == AMC_BF16;
  int rc = make_tmap_4d_16(&map[0], p.k, bf16, p.batch, 2 * p.kv_heads, p.nk, p.d, p.ks, 16);
  if (!rc) rc = make_tmap_4d_16(&map[1], p.v, bf16, p.batch, p.kv_heads, p.nk, p.dv, p.vs, 16);
  if (rc == AMC_ERR_UNSUPPORTED) return AMC_OK;
  if (rc) return rc;
  *handled = true;
  SplitArgs a = plan(p);
  a.part_ml = (float2*)p.workspace;
  a.part = (float*)(a.part_ml + kPartRows);
  if (bf16) return p.dv <= 64 ? split_launch<__nv_bfloat16, 64>(p, a, map, s) : split_launch<__nv_bfloat16, 128>(p, a, map, s);
  return p.dv <= 64 ? split_launch<__half, 64>(p, a, map, s) : split_launch<__half, 128>(p, a, map, s);
}

int diff_split_check_error() {
  int e = 0;
  AMC_CUDA(cudaMemcpyFromSymbol(&e, g_diff_split_error, sizeof(int)));
  if (e) {
    int z = 0;
    AMC_CUDA(cudaMemcpyToSymbol(g_diff_split_error, &z, sizeof(int)));
    return fail(e, "diff_attention: a bounded wait of the single-token form gave up");
  }
  return AMC_OK;
}

}  // namespace amc
