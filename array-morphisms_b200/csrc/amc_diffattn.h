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

// Per (batch, head, row) of the backward: both maps' lse * log2 e (+inf where
// the row is empty, so that exp2(s - lse) is 0) and D = rowsum(dO * O_m).
struct DiffRow {
  float lse1, d1, lse2, d2;
};

// Workspace of the backward: DiffRow rows, then one partial of dlam per
// (head, batch, row tile of kDiffTile).
constexpr int kDiffTile = 32;
inline size_t diff_rows_bytes(const amc_diff_attention& p) {
  return (size_t)p.batch * p.heads * p.nq * sizeof(DiffRow);
}
inline size_t diff_partials(const amc_diff_attention& p) {
  return (size_t)p.batch * p.heads * ((p.nq + kDiffTile - 1) / kDiffTile);
}

// Tensor-core forward; *handled = false (and nothing launched) for other
// types, shapes and alignments.
bool diff_tc_shape(const amc_diff_attention& p);
int diff_fwd_tc(const amc_diff_attention& p, cudaStream_t s, bool* handled);
int launch_diff_fwd_simt(const amc_diff_attention& p, cudaStream_t s);
int launch_diff_bwd_simt(const amc_diff_attention& p, DiffRow* rows, float* partials, cudaStream_t s);
int launch_diff_bwd_rows(const amc_diff_attention& p, DiffRow* rows, cudaStream_t s);
// tiles: partials per (head, batch)
int launch_diff_dlam(const amc_diff_attention& p, const float* partials, int tiles, cudaStream_t s);

}  // namespace amc
