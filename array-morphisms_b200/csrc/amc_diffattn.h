// Shared by the differential-attention translation units.
#pragma once

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

// Workspace of the backward.  For every two rows (2 r, 2 r + 1) of a (batch,
// head) one float4 of each kind, negated for the fused operations that use
// them, both rows of map 1 and then both of map 2:
//   nlse = -lse * log2 e, -inf where the row is empty, so that
//          exp2(s + nlse) is 0
//   nsum = -D_m, D_m = rowsum(dO * O_m)
// (rows padded to a multiple of 4, so that a tile of them is a bulk copy),
// then lam of every head, then one partial of sum P_2 G for every (head,
// batch, row tile).
constexpr int kDiffTile = 32;
struct DiffBwdWork {
  float4* nlse;
  float4* nsum;
  float* lam;
  float* partials;
  int pitch;   // rows of a (batch, head)
};
// The value of row r of map m in such an array.
__device__ __forceinline__ float diff_row(const float4* x, int64_t first_row, int r, int m) {
  return reinterpret_cast<const float*>(x + (first_row + r) / 2)[2 * m + (r & 1)];
}
inline int diff_row_pitch(const amc_diff_attention& p) { return (p.nq + 3) & ~3; }
inline size_t diff_bwd_bytes(const amc_diff_attention& p) {
  const size_t rows = (size_t)p.batch * p.heads * diff_row_pitch(p);
  const size_t partials = (size_t)p.batch * p.heads * ((p.nq + kDiffTile - 1) / kDiffTile);
  return rows * sizeof(float4) + (size_t)p.heads * sizeof(float) + partials * sizeof(float);
}
inline DiffBwdWork diff_bwd_work(const amc_diff_attention& p) {
  const size_t rows = (size_t)p.batch * p.heads * diff_row_pitch(p);
  DiffBwdWork w;
  w.nlse = (float4*)p.workspace;
  w.nsum = w.nlse + rows / 2;
  w.lam = (float*)(w.nsum + rows / 2);
  w.partials = w.lam + p.heads;
  w.pitch = diff_row_pitch(p);
  return w;
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
// Tensor-core gradients (after the rows), likewise.
int diff_bwd_tc(const amc_diff_attention& p, const DiffBwdWork& w, cudaStream_t s, bool* handled);
// tiles: partials per (head, batch)
int launch_diff_dlam(const amc_diff_attention& p, const DiffBwdWork& w, int tiles, cudaStream_t s);

}  // namespace amc
