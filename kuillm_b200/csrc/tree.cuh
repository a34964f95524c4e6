// Argument blocks shared by the kernels that work on a KV cache across decode steps: attention of drafted
// tokens (sdpa_tree*.cu) and the attention weight a key has received (attn_mass*.cu).
#pragma once
#include "common.cuh"

namespace kuiops {

// The argument blocks of the C ABI (include/kuiops.h) are what the kernels take.
using TreeArgs = kuiops_sdpa_tree_args;
using MassArgs = kuiops_attn_mass_args;

// Division of a 31-bit number by a launch constant: q = (umulhi(n, mul) + n) >> shift with 2^(shift - 1) < d <= 2^shift
// and mul = floor(2^32 (2^shift - d) / d) + 1 (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994).  The hardware has no integer division, and the
// sequence that stands for it costs more than most of what these kernels do per item.
struct FastDiv {
  uint32_t d, mul, shift;
  void set(uint32_t v) {
    d = v;
    for (shift = 0; (1ull << shift) < v; ++shift) {}
    mul = uint32_t((((1ull << shift) - v) << 32) / v + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

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

// The tensor-core kernel, with its own joining; the workspace it needs does not depend on pointers and strides.
bool sdpa_tree_tc_eligible(const TreeArgs& a);
size_t sdpa_tree_tc_workspace_bytes(const TreeArgs& a);
int sdpa_tree_tc(const TreeArgs& a, cudaStream_t st);

int attn_mass_simt(const MassArgs& a, cudaStream_t st);
bool attn_mass_tc_eligible(const MassArgs& a);
int attn_mass_tc(const MassArgs& a, cudaStream_t st);

__device__ __forceinline__ uint32_t clamp_len(long long v, uint32_t s) {
  return v < 0 ? 0u : (v < (long long)s ? uint32_t(v) : s);
}

}  // namespace kuiops
