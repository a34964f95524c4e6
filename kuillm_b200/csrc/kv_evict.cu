// Eviction from a KV cache by accumulated attention weight.  Per (batch, KV head) row of kv_lens[b] slots the `budget`
// slots with the most weight stay (protected slots before all others; equal weights: the lower slot).  The cache is not
// repacked: the i-th evicted slot below the budget takes over the i-th kept slot at or above it, so only that many rows
// of K and V move, sources and destinations are disjoint, and every move is independent of the others.
//
// Two launches.  The first finds, per row, the budget-th largest key by radix selection and writes the slot map; the
// second moves the rows of K and V with the whole GPU.
#include "common.cuh"

namespace kuiops {

static_assert(sizeof(kuiops_kv_evict_args) == 184, "callers pack the block without padding");

constexpr int kEvictThreads = 1024;
constexpr int kEvictWarps = kEvictThreads / 32;

struct EvictArgs : kuiops_kv_evict_args {
  int32_t *holes, *movers, *moves;      // in the workspace: per row up to `pairs` (hole, mover) slots, and their number
  uint32_t pairs;
  int wide;                             // every row of K and V starts on a 16-byte boundary and is whole vectors
};

// Order-preserving image of a slot's weight: NaN above +inf, protected slots above all.
__device__ __forceinline__ uint32_t evict_key(float w, bool held) {
  if (held) return 0xFFFFFFFFu;
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t u = __float_as_uint(w + 0.f);           // -0 counts as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct EvictRow {
  const float* mass; const int32_t* pos;
  long long recent_from;                // positions from here on are protected
  uint32_t sinks;
  __device__ __forceinline__ uint32_t key(uint32_t i) const {
    const long long ps = pos ? (long long)pos[i] : (long long)i;
    return evict_key(mass[i], (ps >= 0 && ps < (long long)sinks) || ps >= recent_from);
  }
};

// Exclusive prefix over the warps of the CTA of a per-warp count; `buf` holds kEvictWarps words.  Every thread of warp w
// gets the sum of the warps before w.
__device__ __forceinline__ uint32_t warp_prefix(uint32_t count, uint32_t* buf, uint32_t* total) {
  const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) buf[w] = count;
  __syncthreads();
  uint32_t v = buf[lane], t = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= uint32_t(o)) t += x;
  }
  *total = __shfl_sync(0xffffffffu, t, 31);
  return __shfl_sync(0xffffffffu, t - v, w);
}

__global__ void __launch_bounds__(kEvictThreads)
kv_evict_select_kernel(const EvictArgs p) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t wbuf[kEvictWarps];
  __shared__ uint32_t s_prefix, s_need;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t row = blockIdx.x, b = row / p.h_kv, g = b % p.lens_n;
  pdl_wait();
  pdl_trigger();
  const long long len64 = p.kv_lens[g];
  const uint32_t len = len64 < 0 ? 0u : (len64 < (long long)p.cap ? uint32_t(len64) : p.cap);
  const uint32_t kept = min(len, p.budget);
  const size_t at = size_t(row) * p.cap;
  EvictRow r;
  r.mass = p.mass + at; r.pos = p.pos ? p.pos + at : nullptr; r.sinks = p.sinks;
  r.recent_from = (p.next_pos ? (long long)p.next_pos[g] : (long long)len) - (long long)p.recent;
  int32_t* src = p.src + size_t(row) * p.budget;
  if (tid == 0 && row % p.h_kv == 0 && b < p.lens_n) p.lens_out[g] = kept;

  uint32_t moved = 0;
  int32_t* holes = p.holes + size_t(row) * p.pairs;
  int32_t* movers = p.movers + size_t(row) * p.pairs;
  if (len > p.budget) {
    // radix selection, eight bits a pass: `prefix` collects the digits of the budget-th largest key, `need` its rank
    // among the keys that share the digits found so far
    uint32_t prefix = 0, need = p.budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (uint32_t i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t himask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
      for (uint32_t i = tid; i < len; i += kEvictThreads) {
        const uint32_t k = r.key(i);
        if ((k & himask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (warp == 0) {
        // lane x holds bins 8 x .. 8 x + 7; counts of the bins above, from the top
        uint32_t c[8], sum = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) { c[x] = hist[lane * 8 + x]; sum += c[x]; }
        uint32_t suffix = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t v = __shfl_down_sync(0xffffffffu, suffix, o);
          if (lane + o < 32) suffix += v;
        }
        uint32_t above = suffix - sum;
#pragma unroll
        for (int x = 7; x >= 0; --x) {
          if (above < need && above + c[x] >= need) { s_prefix = prefix | ((lane * 8 + x) << shift); s_need = need - above; }
          above += c[x];
        }
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
    }
    // keys above `prefix` stay, and the first `need` slots of those equal to it.  A warp owns a contiguous run of slots.
    const uint32_t run = ((len + kEvictWarps - 1) / kEvictWarps + 31) & ~31u;
    const uint32_t lo = min(warp * run, len), hi = min(lo + run, len);
    uint32_t total, ties = 0;
    for (uint32_t i = lo; i < hi; i += 32)
      ties += __popc(__ballot_sync(0xffffffffu, i + lane < hi && r.key(i + lane) == prefix));
    const uint32_t ties_before = warp_prefix(ties, wbuf, &total);
    uint32_t n_hole = 0, n_move = 0, hole_base = 0, move_base = 0;
    for (int pass = 0; pass < 2; ++pass) {
      uint32_t t = ties_before, nh = 0, nm = 0;
      for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
        const uint32_t i = i0 + lane;
        const bool in = i < hi;
        const uint32_t k = in ? r.key(i) : 0u;
        const uint32_t eq = __ballot_sync(0xffffffffu, in && k == prefix);
        const uint32_t below = (1u << lane) - 1u;
        const bool keep = in && (k > prefix || (k == prefix && t + __popc(eq & below) < need));
        t += __popc(eq);
        const uint32_t hb = __ballot_sync(0xffffffffu, in && !keep && i < p.budget);
        const uint32_t mb = __ballot_sync(0xffffffffu, keep && i >= p.budget);
        if (pass == 1) {
          if (in && !keep && i < p.budget) holes[hole_base + nh + __popc(hb & below)] = int32_t(i);
          if (keep && i >= p.budget) movers[move_base + nm + __popc(mb & below)] = int32_t(i);
          if (keep && i < p.budget) {
            src[i] = int32_t(i);
            p.mass_out[at + i] = r.mass[i];
            p.pos_out[at + i] = r.pos ? r.pos[i] : int32_t(i);
          }
        }
        nh += __popc(hb); nm += __popc(mb);
      }
      if (pass == 0) {
        hole_base = warp_prefix(nh, wbuf, &n_hole);
        move_base = warp_prefix(nm, wbuf, &n_move);
      }
    }
    moved = n_move;                     // = n_hole: as many slots are kept as there are below the budget
    __syncthreads();                    // the lists (global memory, this CTA's own) are complete
    for (uint32_t i = tid; i < moved; i += kEvictThreads) {
      const int32_t to = holes[i], from = movers[i];
      src[to] = from;
      p.mass_out[at + to] = r.mass[from];
      p.pos_out[at + to] = r.pos ? r.pos[from] : from;
    }
  } else {
    for (uint32_t i = tid; i < len; i += kEvictThreads) {
      src[i] = int32_t(i);
      p.mass_out[at + i] = r.mass[i];
      p.pos_out[at + i] = r.pos ? r.pos[i] : int32_t(i);
    }
  }
  for (uint32_t i = kept + tid; i < p.budget; i += kEvictThreads) src[i] = -1;
  for (uint32_t i = kept + tid; i < p.cap; i += kEvictThreads) { p.mass_out[at + i] = 0.f; p.pos_out[at + i] = -1; }
  if (tid == 0) p.moves[row] = int32_t(moved);
}

// blockIdx.x: row * parts + part.  A warp moves one slot's K row and V row at a time.
__global__ void __launch_bounds__(256)
kv_evict_move_kernel(const EvictArgs p, uint32_t parts) {
  const uint32_t row = blockIdx.x / parts, part = blockIdx.x % parts;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const uint32_t moved = uint32_t(p.moves[row]);
  const uint32_t b = row / p.h_kv, kvh = row % p.h_kv;
  const int32_t* holes = p.holes + size_t(row) * p.pairs;
  const int32_t* movers = p.movers + size_t(row) * p.pairs;
  char* K = static_cast<char*>(p.K) + (int64_t(b) * p.k_sn + int64_t(kvh) * p.k_sh) * p.elem_bytes;
  char* V = static_cast<char*>(p.V) + (int64_t(b) * p.v_sn + int64_t(kvh) * p.v_sh) * p.elem_bytes;
  const int64_t ks = p.k_ss * p.elem_bytes, vs = p.v_ss * p.elem_bytes;
  const uint32_t kb = p.e * p.elem_bytes, vb = p.ev * p.elem_bytes, unit = p.wide ? 16 : p.elem_bytes;
  for (uint32_t i = part * 8 + warp; i < moved; i += parts * 8) {
    const int64_t to = holes[i], from = movers[i];
    for (uint32_t c = lane * unit; c < kb; c += 32 * unit) {
      if (unit == 16) *reinterpret_cast<int4*>(K + to * ks + c) = *reinterpret_cast<const int4*>(K + from * ks + c);
      else if (unit == 4) *reinterpret_cast<uint32_t*>(K + to * ks + c) = *reinterpret_cast<const uint32_t*>(K + from * ks + c);
      else if (unit == 2) *reinterpret_cast<uint16_t*>(K + to * ks + c) = *reinterpret_cast<const uint16_t*>(K + from * ks + c);
      else K[to * ks + c] = K[from * ks + c];
    }
    for (uint32_t c = lane * unit; c < vb; c += 32 * unit) {
      if (unit == 16) *reinterpret_cast<int4*>(V + to * vs + c) = *reinterpret_cast<const int4*>(V + from * vs + c);
      else if (unit == 4) *reinterpret_cast<uint32_t*>(V + to * vs + c) = *reinterpret_cast<const uint32_t*>(V + from * vs + c);
      else if (unit == 2) *reinterpret_cast<uint16_t*>(V + to * vs + c) = *reinterpret_cast<const uint16_t*>(V + from * vs + c);
      else V[to * vs + c] = V[from * vs + c];
    }
  }
}

static uint32_t evict_pairs(uint32_t cap, uint32_t budget) {
  if (budget >= cap) return 0;
  return budget < cap - budget ? budget : cap - budget;
}

}  // namespace kuiops

using namespace kuiops;

extern "C" {

size_t kuiops_kv_evict_workspace_bytes(uint32_t n, uint32_t h_kv, uint32_t cap, uint32_t budget) {
  return size_t(n) * h_kv * 4 * (2 * size_t(evict_pairs(cap, budget)) + 1);
}

int kuiops_kv_evict(const kuiops_kv_evict_args* args, kuiops_stream_t stream) {
  if (!args) return KUIOPS_EINVAL;
  EvictArgs a = {};
  static_cast<kuiops_kv_evict_args&>(a) = *args;
  const uint32_t elem_bytes = a.elem_bytes, n = a.n, h_kv = a.h_kv, e = a.e, ev = a.ev;
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return KUIOPS_EINVAL;
  if (n == 0 || h_kv == 0 || a.cap == 0 || e == 0 || ev == 0 || a.budget == 0 || a.lens_n == 0 || n % a.lens_n) return KUIOPS_EINVAL;
  if (!a.K || !a.V || !a.mass || !a.kv_lens || !a.mass_out || !a.pos_out || !a.src || !a.lens_out) return KUIOPS_EINVAL;
  if (a.mass_out == a.mass || a.pos_out == a.pos || a.lens_out == a.kv_lens || a.k_ss < int64_t(e) || a.v_ss < int64_t(ev)) return KUIOPS_EINVAL;
  if (a.budget > a.cap || uint64_t(a.sinks) + a.recent > a.budget) return KUIOPS_EINVAL;
  if (a.cap > 0x7fffff00u || uint64_t(n) * h_kv >= (1ull << 31) || uint64_t(e > ev ? e : ev) * 4 >= (1ull << 31)) return KUIOPS_ELIMIT;
  if (!a.workspace || a.workspace_bytes < kuiops_kv_evict_workspace_bytes(n, h_kv, a.cap, a.budget) ||
      (reinterpret_cast<uintptr_t>(a.workspace) & 3))
    return KUIOPS_EWORKSPACE;
  const uint32_t rows = n * h_kv;
  a.pairs = evict_pairs(a.cap, a.budget);
  a.moves = static_cast<int32_t*>(a.workspace);
  a.holes = a.moves + rows;
  a.movers = a.holes + size_t(rows) * a.pairs;
  auto whole = [&](const void* t, uint32_t f, int64_t sn, int64_t sh, int64_t sl) {
    const int64_t v = 16 / elem_bytes;
    return aligned16(t) && f % v == 0 && (n == 1 || sn % v == 0) && (h_kv == 1 || sh % v == 0) && sl % v == 0;
  };
  a.wide = whole(a.K, e, a.k_sn, a.k_sh, a.k_ss) && whole(a.V, ev, a.v_sn, a.v_sh, a.v_ss);
  cudaStream_t st = as_stream(stream);
  const int rc = launch_pdl(kv_evict_select_kernel, dim3(rows), dim3(kEvictThreads), 0, st, a);
  if (rc != KUIOPS_OK || a.pairs == 0) return rc;
  const uint64_t want = (uint64_t(a.pairs) + 63) / 64, most = (16ull * num_sms() + rows - 1) / rows;
  const uint32_t parts = uint32_t(want < most ? want : most);
  if (uint64_t(rows) * parts >= (1ull << 31)) return KUIOPS_ELIMIT;
  return launch_pdl(kv_evict_move_kernel, dim3(rows * parts), dim3(256), 0, st, a, parts);
}

}  // extern "C"
