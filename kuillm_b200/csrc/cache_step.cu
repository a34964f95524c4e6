// What follows the verification of a tree of drafted tokens: the greedy walk through it (kuiops_tree_accept) and the
// commit of the accepted rows to the cache (kuiops_kv_append).  Both are bound by launch latency at decode sizes
// (replayed from a graph: the walk of 8 nodes 2.2 us, of 256 sequences with 255 nodes 4.2 us; one committed token 2.3 us, 16 sequences in 32
// layers 9.2 us: a warp copies its K row and then its V row, one load under way at a time, and waits for memory at each).
#include "common.cuh"

namespace kuiops {

static_assert(sizeof(kuiops_tree_accept_args) == 72, "callers pack the block without padding");
static_assert(sizeof(kuiops_kv_append_args) == 224, "callers pack the block without padding");

constexpr int kAcceptThreads = 128;

// One CTA per sequence.  Node i is accepted when every node j on its way to the root (itself included, the root not)
// has draft[j] == target[parent[j]]; the deepest accepted node wins, the lowest index among equals.
__global__ void __launch_bounds__(kAcceptThreads)
tree_accept_kernel(uint32_t l, const int64_t* __restrict__ parents, int64_t par_sn, const int64_t* __restrict__ draft,
                   const int64_t* __restrict__ target, int64_t* __restrict__ path, int64_t* __restrict__ counts,
                   int64_t* __restrict__ next, int32_t* status) {
  extern __shared__ int sh[];
  int* up = sh;                         // parent, or -1 where the chain breaks
  __shared__ unsigned long long best;
  const uint32_t b = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const int64_t* par = parents + int64_t(b) * par_sn;
  const int64_t* dr = draft + size_t(b) * l;
  const int64_t* tg = target + size_t(b) * l;
  if (threadIdx.x == 0) best = 0;
  for (uint32_t i = threadIdx.x; i < l; i += kAcceptThreads) {
    const long long p = par[i];
    const bool child = i > 0 && p >= 0 && p < (long long)i;
    if (status && (i == 0 ? p >= 0 : p >= (long long)i)) *status = 1;       // the root has no parent; a parent comes first
    up[i] = child && dr[i] == tg[p] ? int(p) : -1;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < l; i += kAcceptThreads) {
    uint32_t depth = 1;
    int cur = int(i);
    while (cur > 0) { cur = up[cur]; ++depth; }      // parents have smaller indices: ends after at most i steps
    if (cur == 0) atomicMax(&best, (static_cast<unsigned long long>(depth) << 32) | uint32_t(~i));
  }
  __syncthreads();
  const uint32_t depth = uint32_t(best >> 32);
  int64_t* out = path + size_t(b) * l;
  for (uint32_t i = depth + threadIdx.x; i < l; i += kAcceptThreads) out[i] = -1;
  if (threadIdx.x == 0) {
    int cur = int(~uint32_t(best));
    next[b] = tg[cur];
    counts[b] = depth;
    for (uint32_t t = depth; t-- > 0; cur = up[cur]) out[t] = cur;
  }
}

using AppendArgs = kuiops_kv_append_args;

__device__ __forceinline__ void copy_row(const char* src, char* dst, uint32_t bytes, uint32_t elem, int wide, uint32_t lane) {
  if (wide) {
    for (uint32_t i = lane * 16; i < bytes; i += 512) *reinterpret_cast<int4*>(dst + i) = *reinterpret_cast<const int4*>(src + i);
  } else if (elem == 4) {
    for (uint32_t i = lane * 4; i < bytes; i += 128) *reinterpret_cast<uint32_t*>(dst + i) = *reinterpret_cast<const uint32_t*>(src + i);
  } else if (elem == 2) {
    for (uint32_t i = lane * 2; i < bytes; i += 64) *reinterpret_cast<uint16_t*>(dst + i) = *reinterpret_cast<const uint16_t*>(src + i);
  } else {
    for (uint32_t i = lane; i < bytes; i += 32) dst[i] = src[i];
  }
}

// blockIdx.x: batch entry * parts + part.  A warp moves one accepted row of one KV head (K, then V) at a time.
__global__ void __launch_bounds__(256)
kv_append_kernel(const AppendArgs p, uint32_t parts, int wide) {
  const uint32_t b = blockIdx.x / parts, part = blockIdx.x % parts, g = b % p.lens_n;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const long long len = p.kv_lens[g];
  long long cnt = p.counts ? p.counts[g] : (long long)p.l;
  cnt = cnt < 0 ? 0 : (cnt > (long long)p.l ? (long long)p.l : cnt);
  if (b < p.lens_n && part == 0 && threadIdx.x == 0 && p.lens_out) {
    const long long to = len + cnt;
    p.lens_out[g] = to > (long long)p.cap ? (long long)p.cap : to;
  }
  const uint32_t items = uint32_t(cnt) * p.h_kv;
  for (uint32_t it = part * 8 + warp; it < items; it += parts * 8) {
    const uint32_t kvh = it % p.h_kv, t = it / p.h_kv;
    const long long row = p.path ? p.path[size_t(g) * p.l + t] : (long long)t;
    const long long slot = len + t;
    if (row < 0 || row >= (long long)p.l || slot < 0 || slot >= (long long)p.cap) {
      if (p.status && lane == 0) *p.status = 1;
      continue;
    }
    const uint32_t eb = p.elem_bytes;
    copy_row(static_cast<const char*>(p.DK) + (int64_t(b) * p.dk_sn + int64_t(kvh) * p.dk_sh + row * p.dk_sl) * eb,
             static_cast<char*>(p.K) + (int64_t(b) * p.k_sn + int64_t(kvh) * p.k_sh + slot * p.k_ss) * eb, p.e * eb, eb, wide, lane);
    copy_row(static_cast<const char*>(p.DV) + (int64_t(b) * p.dv_sn + int64_t(kvh) * p.dv_sh + row * p.dv_sl) * eb,
             static_cast<char*>(p.V) + (int64_t(b) * p.v_sn + int64_t(kvh) * p.v_sh + slot * p.v_ss) * eb, p.ev * eb, eb, wide, lane);
    if (lane == 0) {
      const size_t at = (size_t(b) * p.h_kv + kvh) * p.cap + size_t(slot);
      if (p.pos) p.pos[at] = int32_t(p.next_pos[g] + t);
      if (p.mass) p.mass[at] = 0.f;
    }
  }
}

}  // namespace kuiops

using namespace kuiops;

extern "C" {

int kuiops_tree_accept(const kuiops_tree_accept_args* args, kuiops_stream_t stream) {
  if (!args) return KUIOPS_EINVAL;
  const kuiops_tree_accept_args& a = *args;
  if (a.n == 0 || a.l == 0 || !a.parents || !a.draft || !a.target || !a.path || !a.counts || !a.next) return KUIOPS_EINVAL;
  if (a.parents_sn != 0 && a.parents_sn < int64_t(a.l)) return KUIOPS_EINVAL;
  if (a.l > KUIOPS_TREE_MAX_ROWS || a.n >= (1u << 31)) return KUIOPS_ELIMIT;
  return launch_pdl(tree_accept_kernel, dim3(a.n), dim3(kAcceptThreads), size_t(a.l) * 4, as_stream(stream), a.l, a.parents, a.parents_sn, a.draft,
                    a.target, a.path, a.counts, a.next, a.status);
}

int kuiops_kv_append(const kuiops_kv_append_args* args, kuiops_stream_t stream) {
  if (!args) return KUIOPS_EINVAL;
  const AppendArgs& a = *args;
  const uint32_t elem_bytes = a.elem_bytes, n = a.n, h_kv = a.h_kv, l = a.l, e = a.e, ev = a.ev;
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return KUIOPS_EINVAL;
  if (n == 0 || h_kv == 0 || l == 0 || a.cap == 0 || e == 0 || ev == 0 || a.lens_n == 0 || n % a.lens_n) return KUIOPS_EINVAL;
  if (!a.DK || !a.DV || !a.K || !a.V || !a.kv_lens || (a.pos && !a.next_pos)) return KUIOPS_EINVAL;
  if (a.dk_sl < int64_t(e) || a.dv_sl < int64_t(ev) || a.k_ss < int64_t(e) || a.v_ss < int64_t(ev)) return KUIOPS_EINVAL;
  if (a.cap > 0x7fffff00u || uint64_t(l) * h_kv >= (1ull << 31) || uint64_t(e > ev ? e : ev) * 4 >= (1ull << 31)) return KUIOPS_ELIMIT;
  auto whole = [&](const void* t, uint32_t f, int64_t sn, int64_t sh, int64_t sl) {
    const int64_t v = 16 / elem_bytes;
    return aligned16(t) && f % v == 0 && (n == 1 || sn % v == 0) && (h_kv == 1 || sh % v == 0) && sl % v == 0;
  };
  // every row of all four tensors starts on a 16-byte boundary and is whole vectors
  const int wide = whole(a.DK, e, a.dk_sn, a.dk_sh, a.dk_sl) && whole(a.DV, ev, a.dv_sn, a.dv_sh, a.dv_sl) &&
                   whole(a.K, e, a.k_sn, a.k_sh, a.k_ss) && whole(a.V, ev, a.v_sn, a.v_sh, a.v_ss);
  // one CTA per 64 rows that could be accepted: those that are not cost a look at the count
  const uint64_t parts64 = (uint64_t(l) * h_kv + 63) / 64;
  const uint32_t parts = uint32_t(parts64 > 16 ? 16 : parts64);
  if (uint64_t(n) * parts >= (1ull << 31)) return KUIOPS_ELIMIT;
  return launch_pdl(kv_append_kernel, dim3(n * parts), dim3(256), 0, as_stream(stream), a, parts, wide);
}

}  // extern "C"
