// Differential attention of few rows over many keys (the single-token form),
// 16-bit tensors with d <= 64 and dv <= 128, both multiples of 8.
//
// The bound is HBM: every key and value is read once, for all rows (query
// heads that share the key head, times their rows) of a 16-row block.  The
// keys of one sequence and key head are cut into chunks, one CTA each, and
// within a chunk its four warps take every fourth block of 16 keys.  Warps do
// not wait for each other: each has its own ring of TMA boxes (K_1, K_2 and V
// rows of 16 keys, 8 KB), its own running maximum, sum and output, and they
// meet at the end of the chunk in shared memory.  The products are
// mma.sync m16n8k16: 16 rows fill a legacy tile, where a tcgen05 tile of 128
// would be an eighth full, and at 16 rows they take less than half the time
// of the loads.  P is taken into P V as the sum of two 16-bit values (the
// rounded one and the rounding's remainder), which the loads hide: the result
// carries no rounding of P.  A second kernel joins the chunks' outputs by
// their maxima and sums; with one chunk the first kernel writes the result.
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
constexpr int kMinChunk = 256;       // keys: 4 boxes a warp
constexpr int kTargetCtas = 148 * 8; // chunks at full lengths: enough that sequences of different lengths even out
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994530942f;

__device__ int g_diff_split_error;

struct SplitArgs {
  int group, row_blocks, splits, chunk;
  float* part;       // [unit][split][row][map][dv] unscaled outputs
  float2* part_ml;   // [unit][split][row][map] maximum (log2 units) and sum
};

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

template <typename T, int NV>
__global__ void __launch_bounds__(kWarps * 32) k_diff_split(const __grid_constant__ CUtensorMap mK,
                                                           const __grid_constant__ CUtensorMap mV,
                                                           const __grid_constant__ amc_diff_attention p,
                                                           const __grid_constant__ SplitArgs a) {
  constexpr int NT = NV / 8;
  extern __shared__ unsigned char diff_sm_raw[];
  unsigned char* sm = (unsigned char*)(((uintptr_t)diff_sm_raw + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, pos = lane & 3;
  uint64_t* full = (uint64_t*)(sm + kStageBytes) + warp * kStages;
  volatile int* failed = (volatile int*)(sm + kStageBytes + 256);
  const int unit = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int rb = unit % a.row_blocks, g = unit / a.row_blocks % p.kv_heads, b = unit / a.row_blocks / p.kv_heads;
  const int rows = min(kRows, a.group * p.nq - rb * kRows);
  const DiffLens len = diff_lens(p, b);
  int kmax = 0;   // keys that any row of the block sees
  int lim[2];     // of this lane's two rows
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int rr = quad + 8 * r;
    int h, i;
    unit_row(p, a, g, rb * kRows + min(rr, rows - 1), h, i);
    lim[r] = rr < rows ? diff_limit(len, p.causal, i) : 0;
    kmax = max(kmax, lim[r]);
  }
#pragma unroll
  for (int o = 16; o >= 4; o >>= 1) kmax = max(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
  const int kbeg = split * a.chunk, kend = min(kmax, kbeg + a.chunk);
  // box n of this warp starts at key kbeg + 16 (warp + 4 n)
  const int boxes = kend > kbeg ? (kend - kbeg + 15) / 16 : 0;
  const int mine = boxes > warp ? (boxes - warp + kWarps - 1) / kWarps : 0;
  unsigned char* ring = sm + warp * kStages * kBox;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    if (warp == 0) *failed = 0;
    mbar_fence_init();
  }
  __syncthreads();
  auto load = [&](int n) {
    unsigned char* st = ring + n % kStages * kBox;
    const int key = kbeg + 16 * (warp + kWarps * n);
    mbar_expect_tx(&full[n % kStages], 4096 + NV / 64 * 2048);
    tma_load_4d(st, &mK, 0, key, 2 * g, b, &full[n % kStages]);
    tma_load_4d(st + 2048, &mK, 0, key, 2 * g + 1, b, &full[n % kStages]);
    for (int c = 0; c < NV / 64; ++c) tma_load_4d(st + 4096 + c * 2048, &mV, 64 * c, key, g, b, &full[n % kStages]);
  };
  if (lane == 0)
    for (int n = 0; n < kStages && n < mine; ++n) load(n);
  // Q fragments: rows quad and quad + 8, columns 16 k + 2 pos (+8)
  uint32_t q[2][4][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      int h, i;
      unit_row(p, a, g, rb * kRows + min(quad + 8 * r, rows - 1), h, i);
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
  float top[2][2], sum[2][2], o[2][NT][4];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    top[m][0] = top[m][1] = -INFINITY;
    sum[m][0] = sum[m][1] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
  }
  const int mrow = lane & 7, mid = lane >> 3;   // ldmatrix: row and matrix of this lane's address
  bool ok = true;
  for (int n = 0; n < mine; ++n) {
    unsigned char* st = ring + n % kStages * kBox;
    const int key = kbeg + 16 * (warp + kWarps * n);
    ok = __all_sync(0xffffffffu, mbar_wait(&full[n % kStages], (uint32_t)(n / kStages) & 1u));
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
    uint32_t ph[2][4], pl[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float s[2][4] = {};
      const uint32_t kb = smem_addr(st + m * 2048) + (mrow + (mid >> 1) * 8) * 128;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t f[4];
        ldsm4(f, kb + (((2 * k + (mid & 1)) ^ mrow) << 4));
        mma16<T>(s[0], q[m][k], f[0], f[1]);
        mma16<T>(s[1], q[m][k], f[2], f[3]);
      }
      if (key + 16 > min(lim[0], lim[1])) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key + 8 * t + 2 * pos + (e & 1) >= lim[e >> 1]) s[t][e] = -INFINITY;
      }
      bool up = false;
      float mt[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        mt[r] = x * c2;
        up = up || mt[r] > top[m][r] + 8.f;
      }
      if (__any_sync(0xffffffffu, up)) {
        // raise the maxima that lag by more than 2^8
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool raise = mt[r] > top[m][r] + 8.f;
          const float corr = raise ? ex2_approx(top[m][r] - mt[r]) : 1.f;
          if (raise) top[m][r] = mt[r];
          sum[m][r] *= corr;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            o[m][t][2 * r] *= corr;
            o[m][t][2 * r + 1] *= corr;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float base = top[m][r] == -INFINITY ? 0.f : top[m][r];
          const float p0 = ex2_approx(fmaf(s[t][2 * r], c2, -base)), p1 = ex2_approx(fmaf(s[t][2 * r + 1], c2, -base));
          sum[m][r] += p0 + p1;
          const uint32_t hi = pack2<T>(p0, p1);
          const float2 back = unpack2<T>(hi);
          ph[m][2 * t + r] = hi;
          pl[m][2 * t + r] = pack2<T>(p0 - back.x, p1 - back.y);
        }
    }
#pragma unroll
    for (int t = 0; t < NT / 2; ++t) {
      uint32_t f[4];
      const int chunk = 2 * (t & 3) + (mid >> 1);
      ldsm4_t(f, smem_addr(st + 4096 + (t >> 2) * 2048) + (mrow + (mid & 1) * 8) * 128 + ((chunk ^ mrow) << 4));
#pragma unroll
      for (int m = 0; m < 2; ++m) {
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
      for (int s = 0; s < kStages && s < mine; ++s) mbar_wait(&full[s], 0, 1 << 14);
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
    for (int r = 0; r < 2; ++r) {
      float l = sum[m][r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int row = quad + 8 * r;
      if (pos == 0) xml[(warp * 2 + m) * kRows + row] = make_float2(top[m][r], l);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<float2*>(xo + ((warp * 2 + m) * kRows + row) * NV + 8 * t + 2 * pos) =
            make_float2(o[m][t][2 * r], o[m][t][2 * r + 1]);
    }
  __syncthreads();
  for (int row = warp; row < rows; row += kWarps) {
    int h, i;
    unit_row(p, a, g, rb * kRows + row, h, i);
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
    if (a.splits > 1) {
      const int64_t at = ((int64_t)blockIdx.x * kRows + row) * 2;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (lane == 0) a.part_ml[at + m] = make_float2(mx[m], l[m]);
#pragma unroll
        for (int c = 0; c < NV / 32; ++c)
          if (32 * c + lane < p.dv) a.part[(at + m) * p.dv + 32 * c + lane] = acc[m][c];
      }
    } else {
      const float lam = lam_of<T>(p, h);
      const float f0 = l[0] > 0.f ? 1.f / l[0] : 0.f, f1 = l[1] > 0.f ? 1.f / l[1] : 0.f;
#pragma unroll
      for (int c = 0; c < NV / 32; ++c) {
        const float o1 = acc[1][c] * f1;
        if (32 * c + lane < p.dv) put_result<T>(p, b, h, i, 32 * c + lane, fmaf(-lam, o1, acc[0][c] * f0), o1);
      }
      if (p.lse && lane < 2) {
        const float ll = lane ? l[1] : l[0], mm = lane ? mx[1] : mx[0];
        p.lse[((int64_t)b * 2 * p.heads + 2 * h + lane) * p.nq + i] = ll > 0.f ? fmaf(mm, kLn2, logf(ll)) : -INFINITY;
      }
    }
  }
}

// One CTA per (batch, head, row): its chunks' outputs over their joint maxima.
template <typename T>
__global__ void __launch_bounds__(128) k_diff_join(const __grid_constant__ amc_diff_attention p,
                                                   const __grid_constant__ SplitArgs a) {
  const int i = blockIdx.x % p.nq, h = blockIdx.x / p.nq % p.heads, b = blockIdx.x / p.nq / p.heads;
  const int g = h / a.group, rr = (h - g * a.group) * p.nq + i;
  const int64_t unit = ((int64_t)b * p.kv_heads + g) * a.row_blocks + rr / kRows;
  const DiffLens len = diff_lens(p, b);
  const int n = min(a.splits, (diff_limit(len, p.causal, i) + a.chunk - 1) / a.chunk);   // chunks this row sees
  const float lam = lam_of<T>(p, h);
  const int64_t at0 = (unit * a.splits * kRows + rr % kRows) * 2;
  const int64_t step = kRows * 2;
  float res[2], lse[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    float mx = -INFINITY;
    for (int s = 0; s < n; ++s) mx = fmaxf(mx, a.part_ml[at0 + s * step + m].x);
    const float base = mx == -INFINITY ? 0.f : mx;
    float l = 0.f, acc = 0.f;
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float2 e = a.part_ml[at0 + s * step + m];
      const float f = exp2f(e.x - base);
      l = fmaf(e.y, f, l);
      if (threadIdx.x < p.dv) acc = fmaf(a.part[(at0 + s * step + m) * p.dv + threadIdx.x], f, acc);
    }
    res[m] = l > 0.f ? acc / l : 0.f;
    lse[m] = l > 0.f ? fmaf(mx, kLn2, logf(l)) : -INFINITY;
  }
  if (threadIdx.x < p.dv) put_result<T>(p, b, h, i, threadIdx.x, fmaf(-lam, res[1], res[0]), res[1]);
  if (p.lse && threadIdx.x < 2)
    p.lse[((int64_t)b * 2 * p.heads + 2 * h + threadIdx.x) * p.nq + i] = threadIdx.x ? lse[1] : lse[0];
}

namespace {

SplitArgs plan(const amc_diff_attention& p) {
  SplitArgs a{};
  a.group = p.heads / p.kv_heads;
  a.row_blocks = (int)(((int64_t)a.group * p.nq + kRows - 1) / kRows);
  const int64_t units = (int64_t)p.batch * p.kv_heads * a.row_blocks;
  int64_t want = (kTargetCtas + units - 1) / units;
  const int64_t most = (p.nk + kMinChunk - 1) / kMinChunk;
  if (want > most) want = most;
  if (want < 1) want = 1;
  a.chunk = (int)(((p.nk + want - 1) / want + 63) / 64 * 64);
  a.splits = (p.nk + a.chunk - 1) / a.chunk;
  return a;
}

size_t part_elems(const amc_diff_attention& p, const SplitArgs& a) {
  return (size_t)p.batch * p.kv_heads * a.row_blocks * a.splits * kRows * 2;
}

template <typename T, int NV>
int split_launch(const amc_diff_attention& p, const SplitArgs& a, const CUtensorMap (&map)[2], cudaStream_t s) {
  static std::atomic<uint64_t> attr{0};
  if (int rc = smem_attr_once(k_diff_split<T, NV>, kSplitSmem, attr)) return rc;
  const unsigned grid = (unsigned)((int64_t)p.batch * p.kv_heads * a.row_blocks * a.splits);
  k_diff_split<T, NV><<<grid, kWarps * 32, kSplitSmem, s>>>(map[0], map[1], p, a);
  AMC_CUDA(cudaGetLastError());
  if (a.splits > 1) {
    k_diff_join<T><<<(unsigned)((int64_t)p.batch * p.heads * p.nq), 128, 0, s>>>(p, a);
    AMC_CUDA(cudaGetLastError());
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
  if (!split_shape(p)) return 0;
  const SplitArgs a = plan(p);
  return a.splits > 1 ? part_elems(p, a) * (p.dv * sizeof(float) + sizeof(float2)) : 0;
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
  a.part = (float*)(a.part_ml + part_elems(p, a));
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
