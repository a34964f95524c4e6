// Argument blocks shared by the kernels that work on a KV cache across decode steps: attention of drafted
// tokens (sdpa_tree*.cu) and the attention weight a key has received (attn_mass*.cu).
#pragma once
#include "common.cuh"

namespace kuiops {

struct TreeArgs {
  int dtype;
  uint32_t n, h, h_kv, l, s, e, ev;
  const void* Q; int64_t q_sn, q_sh, q_sl;
  const void* K; int64_t k_sn, k_sh, k_ss;       // cache, s rows per (batch, KV head)
  const void* V; int64_t v_sn, v_sh, v_ss;
  const int64_t* kv_lens;                         // keys of each batch entry in the cache, clamped to [0, s]; NULL: s
  const void* DK; int64_t dk_sn, dk_sh, dk_sl;   // the drafted rows' own keys and values
  const void* DV; int64_t dv_sn, dv_sh, dv_sl;
  const unsigned char* mask; int64_t m_sn;        // [l, l] bytes per batch entry (m_sn = 0: one for all)
  float scale;
  void* out; int64_t o_sn, o_sh, o_sl;
  float* lse;
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

// The tensor-core kernel; sdpa_tree_tc_splits does not depend on pointers and strides.
bool sdpa_tree_tc_eligible(const TreeArgs& a);
uint32_t sdpa_tree_tc_splits(const TreeArgs& a);
int sdpa_tree_tc(const TreeArgs& a, float* partials, cudaStream_t st);

struct MassArgs {
  int dtype;
  uint32_t n, h, h_kv, l, s, e;
  const void* Q; int64_t q_sn, q_sh, q_sl;
  const void* K; int64_t k_sn, k_sh, k_ss;
  const float* lse;                               // (n, h, l)
  const int64_t* kv_lens; uint32_t lens_n;        // entry b reads kv_lens[b % lens_n]; NULL: s
  const int64_t* q_lens;                          // (lens_n, l): leading keys a row counts for; NULL: by is_causal
  float scale;
  int is_causal;
  const float* mass; float* out;                  // (n, h_kv, s); mass NULL: zeros
};

int attn_mass_simt(const MassArgs& a, cudaStream_t st);

__device__ __forceinline__ uint32_t clamp_len(long long v, uint32_t s) {
  return v < 0 ? 0u : (v < (long long)s ? uint32_t(v) : s);
}

}  // namespace kuiops
