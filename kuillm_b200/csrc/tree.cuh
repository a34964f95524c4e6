// Argument blocks shared by the kernels that work on a KV cache across decode steps: attention of drafted
// tokens (sdpa_tree*.cu) and the attention weight a key has received (attn_mass*.cu).
#pragma once
#include "common.cuh"

namespace kuiops {

// The argument blocks of the C ABI (include/kuiops.h) are what the kernels take.
using TreeArgs = kuiops_sdpa_tree_args;
using MassArgs = kuiops_attn_mass_args;

// A parked record of one output row and key slice: ev accumulators (rounded up to 4), maximum (log2 domain), sum, 2 unused.
__host__ __device__ inline uint32_t tree_record_floats(uint32_t ev) { return ((ev + 3) & ~3u) + 4; }
// Record of row (batch, head, position) and slice `split`.
__device__ __forceinline__ float* tree_record(float* partials, uint64_t row, uint32_t splits, uint32_t split, uint32_t ev) {
  return partials + (row * splits + split) * tree_record_floats(ev);
}

// The SIMT kernel: every type, head dimension and stride.
uint32_t sdpa_tree_simt_splits(const TreeArgs& a);
int sdpa_tree_simt(const TreeArgs& a, float* partials, uint32_t splits, cudaStream_t st);
// Joins the records of `splits` slices into out / lse.
int sdpa_tree_merge(const TreeArgs& a, const float* partials, uint32_t splits, cudaStream_t st);

// The tensor-core kernel; sdpa_tree_tc_splits does not depend on pointers and strides.
bool sdpa_tree_tc_eligible(const TreeArgs& a);
uint32_t sdpa_tree_tc_splits(const TreeArgs& a);
int sdpa_tree_tc(const TreeArgs& a, float* partials, cudaStream_t st);

int attn_mass_simt(const MassArgs& a, cudaStream_t st);
bool attn_mass_tc_eligible(const MassArgs& a);
int attn_mass_tc(const MassArgs& a, cudaStream_t st);

__device__ __forceinline__ uint32_t clamp_len(long long v, uint32_t s) {
  return v < 0 ? 0u : (v < (long long)s ? uint32_t(v) : s);
}

}  // namespace kuiops
