// Eviction from a KV cache by accumulated attention weight.  Per (batch, KV head) row of kv_lens[b] slots the `budget`
// slots with the most weight stay (protected slots before all others; equal weights: the lower slot).  The cache is not
// repacked: the i-th evicted slot below the budget takes over the i-th kept slot at or above it, so only that many rows
// of K and V move, sources and destinations are disjoint, and every move is independent of the others.
//
// A thread-block cluster handles a row, every CTA a contiguous slice of its slots, whose order keys it keeps in shared
// memory (the weights are read from HBM once):
//   the budget-th largest key by radix selection, 11 + 11 + 10 bits: every CTA counts its slice, the counts are added over the
//   cluster through distributed shared memory (by every CTA for itself, so nothing is sent back);
//   ties, holes (evicted below the budget) and movers (kept at or above it) are numbered by counts per warp, CTA and cluster;
//   then the rows move, eight pairs of K and V under way per warp: by the cluster's own warps where few can move, else by a second
//   launch that takes the slots from src and spreads them over the whole GPU.
// Bound by the rows it moves (HBM) where many rows move, else by the latency of these steps.
#include "common.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace kuiops {

static_assert(sizeof(kuiops_kv_evict_args) == 168, "callers pack the block without padding");

constexpr int kEvictThreads = 512;        // two CTAs of up to 12288 slots share an SM
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr uint32_t kEvictBins = 2048;
constexpr uint32_t kEvictOwn = kEvictBins / kEvictThreads;      // bins of a thread
constexpr uint32_t kEvictCopies = 2;       // of the first histogram: weights share few exponents, whose bins neighbours in a warp fight for
constexpr uint32_t kEvictMaxCluster = 8;   // the portable cluster size
constexpr uint32_t kEvictMaxKeys = 40960;  // slots of a CTA whose keys fit its shared memory (160 KB); longer slices are read again

struct EvictArgs : kuiops_kv_evict_args {
  uint32_t cached;                         // keys per CTA kept in shared memory: 0 or all of its slice
  int wide;                                // every row of K and V starts on a 16-byte boundary and is whole vectors
};

// Order-preserving image of a slot's weight: NaN above +inf, protected slots above all.
__device__ __forceinline__ uint32_t evict_key(float w, bool held) {
  if (held) return 0xFFFFFFFFu;
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t u = __float_as_uint(w + 0.f);           // -0 counts as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

static_assert(kEvictOwn == 4, "peers' counts are read as one 16-byte word");

struct EvictShared {
  uint32_t hist[3][kEvictBins];            // one per digit: a CTA may still be read by its peers when it starts on the next
  uint32_t copies[kEvictCopies][kEvictBins];
  uint32_t warp_count[2][kEvictWarps];
  uint32_t ties, holes, movers;            // of this CTA's slice, for its peers
  uint32_t bin, need;
};

// Sum of `count` over the warps before this one; *total over all.  `buf`: kEvictWarps words that no other meeting in flight uses.
__device__ __forceinline__ uint32_t warps_before(uint32_t count, uint32_t* buf, uint32_t* total) {
  const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) buf[w] = count;
  __syncthreads();
  const uint32_t v = lane < kEvictWarps ? buf[lane] : 0u;
  uint32_t t = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= uint32_t(o)) t += x;
  }
  *total = __shfl_sync(0xffffffffu, t, 31);
  return __shfl_sync(0xffffffffu, t - v, w);
}

template <int UNIT> struct EvictUnit;
template <> struct EvictUnit<16> { using type = int4; };
template <> struct EvictUnit<4> { using type = uint32_t; };
template <> struct EvictUnit<2> { using type = uint16_t; };
template <> struct EvictUnit<1> { using type = uint8_t; };

// Where a row's K and V lie.
struct EvictRows {
  char *K, *V;
  int64_t ks, vs;
  uint32_t kb, vb;
  __device__ __forceinline__ EvictRows(const EvictArgs& p, uint32_t row) {
    const uint32_t b = row / p.h_kv, kvh = row - b * p.h_kv, eb = p.elem_bytes;
    K = static_cast<char*>(p.K) + (int64_t(b) * p.k_sn + int64_t(kvh) * p.k_sh) * eb;
    V = static_cast<char*>(p.V) + (int64_t(b) * p.v_sn + int64_t(kvh) * p.v_sh) * eb;
    ks = p.k_ss * eb; vs = p.v_ss * eb;
    kb = p.e * eb; vb = p.ev * eb;
  }
};

// The warp moves slots from[x] to to[x] (to[x] < 0: nothing), a row of K and one of V laid end to end, a unit per lane.
template <int UNIT, int N>
__device__ __forceinline__ void move_slots(const EvictRows& r, const int (&to)[N], const int (&from)[N], uint32_t lane) {
  using U = typename EvictUnit<UNIT>::type;
  const uint32_t ku = r.kb / UNIT, units = (r.kb + r.vb) / UNIT;
  for (uint32_t u = lane; u < units; u += 32) {
    char* base = u < ku ? r.K + size_t(u) * UNIT : r.V + size_t(u - ku) * UNIT;
    const int64_t st = u < ku ? r.ks : r.vs;
    U d[N];
#pragma unroll
    for (int x = 0; x < N; ++x)
      if (to[x] >= 0) d[x] = *reinterpret_cast<const U*>(base + from[x] * st);
#pragma unroll
    for (int x = 0; x < N; ++x)
      if (to[x] >= 0) *reinterpret_cast<U*>(base + to[x] * st) = d[x];
  }
}
template <int N>
__device__ __forceinline__ void move_slots(const EvictArgs& p, const EvictRows& r, const int (&to)[N], const int (&from)[N], uint32_t lane) {
  if (p.wide) move_slots<16>(r, to, from, lane);
  else if (p.elem_bytes == 4) move_slots<4>(r, to, from, lane);
  else if (p.elem_bytes == 2) move_slots<2>(r, to, from, lane);
  else move_slots<1>(r, to, from, lane);
}

// The second launch: a warp takes 32 slots below the budget.
__global__ void __launch_bounds__(256)
kv_evict_move_kernel(const EvictArgs p, uint32_t chunks) {
  const uint32_t row = blockIdx.x / chunks, lane = threadIdx.x & 31;
  const uint32_t i0 = ((blockIdx.x - row * chunks) * 8 + (threadIdx.x >> 5)) * 32;
  pdl_wait();
  pdl_trigger();
  const uint32_t i = i0 + lane;
  const int from = i < p.budget ? p.src[size_t(row) * p.budget + i] : -1;
  uint32_t todo = __ballot_sync(0xffffffffu, from >= 0 && from != int(i));
  if (todo == 0) return;
  const EvictRows r(p, row);
  while (todo) {
    constexpr int N = 8;
    int to[N], fr[N];
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int bit = __ffs(todo) - 1;
      fr[x] = __shfl_sync(0xffffffffu, from, bit < 0 ? 0 : bit);
      to[x] = bit < 0 ? -1 : int(i0) + bit;
      todo &= todo - 1;
    }
    move_slots(p, r, to, fr, lane);
  }
}

template <bool MOVES>
__global__ void __launch_bounds__(kEvictThreads, 2)
kv_evict_kernel(const EvictArgs p, uint32_t ctas) {
  extern __shared__ __align__(16) unsigned char raw[];
  EvictShared& sh = *reinterpret_cast<EvictShared*>(raw);
  uint32_t* key_s = reinterpret_cast<uint32_t*>(raw + sizeof(EvictShared));
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t part = ctas > 1 ? cluster.block_rank() : 0, row = blockIdx.x / ctas;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, below = (1u << lane) - 1u;
  const uint32_t b = row / p.h_kv, g = b % p.lens_n;
  pdl_wait();
  pdl_trigger();
  const long long len64 = p.kv_lens[g];
  const uint32_t len = len64 < 0 ? 0u : (len64 < (long long)p.cap ? uint32_t(len64) : p.cap);
  const uint32_t kept = min(len, p.budget);
  const size_t at = size_t(row) * p.cap;
  const float* mass = p.mass + at;
  const int32_t* pos = p.pos ? p.pos + at : nullptr;
  float* mass_out = p.mass_out + at;
  int32_t* pos_out = p.pos_out + at;
  int32_t* src = p.src + size_t(row) * p.budget;
  const long long recent_from = (p.next_pos ? (long long)p.next_pos[g] : (long long)len) - (long long)p.recent;
  if (tid == 0 && part == 0 && row % p.h_kv == 0 && b < p.lens_n) p.lens_out[g] = kept;

  if (len > p.budget) {
    // positions are 32-bit: so are the bounds of the protected ones (sinks <= budget < 2^31; a negative position is no sink)
    const bool some_recent = recent_from <= 0x7fffffffll;
    const int recent32 = recent_from < -0x80000000ll ? int(0x80000000) : int(recent_from);
    auto key_of = [&](uint32_t i) {
      const int ps = pos ? pos[i] : int(i);
      return evict_key(mass[i], uint32_t(ps) < p.sinks || (some_recent && ps >= recent32));
    };
    // this CTA's slots [c_lo, c_hi), this warp's [lo, hi) of them: whole groups of 32
    const uint32_t slice = ((len + ctas - 1) / ctas + 31) & ~31u, c_lo = min(part * slice, len), c_hi = min(c_lo + slice, len);
    const uint32_t run = ((slice + kEvictWarps - 1) / kEvictWarps + 31) & ~31u;
    const uint32_t lo = min(c_lo + warp * run, c_hi), hi = min(lo + run, c_hi);
    const bool cached = p.cached != 0;
    for (uint32_t i = tid; i < kEvictBins; i += kEvictThreads) {
      sh.hist[1][i] = sh.hist[2][i] = 0;
#pragma unroll
      for (uint32_t c = 0; c < kEvictCopies; ++c) sh.copies[c][i] = 0;
    }
    __syncthreads();
    // ---- the budget-th largest key: `prefix` collects its digits, `need` its rank among the keys that share them --------
    uint32_t prefix = 0, need = p.budget;
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      const int shift = d == 0 ? 21 : (d == 1 ? 10 : 0);
      const uint32_t himask = d == 0 ? 0u : 0xFFFFFFFFu << (d == 1 ? 21 : 10), lowmask = d == 2 ? 1023u : 2047u;
      constexpr int B = 8;                 // keys of a thread under way
      for (uint32_t i0 = c_lo + tid; i0 < c_hi; i0 += B * kEvictThreads) {
        uint32_t k[B];
#pragma unroll
        for (int x = 0; x < B; ++x) {
          const uint32_t i = i0 + x * kEvictThreads;
          k[x] = i >= c_hi ? 0u : (d == 0 || !cached ? key_of(i) : key_s[i - c_lo]);
        }
#pragma unroll
        for (int x = 0; x < B; ++x) {
          const uint32_t i = i0 + x * kEvictThreads;
          if (i >= c_hi) break;
          if (d == 0) {
            if (cached) key_s[i - c_lo] = k[x];
            atomicAdd(&sh.copies[lane % kEvictCopies][k[x] >> 21], 1u);
          } else if ((k[x] & himask) == prefix) {
            atomicAdd(&sh.hist[d][(k[x] >> shift) & lowmask], 1u);
          }
        }
      }
      __syncthreads();
      uint32_t c[kEvictOwn];               // this thread's bins, over the cluster
#pragma unroll
      for (uint32_t x = 0; x < kEvictOwn; ++x) {
        const uint32_t bin = kEvictOwn * tid + x;
        if (d == 0) {
          c[x] = 0;
#pragma unroll
          for (uint32_t y = 0; y < kEvictCopies; ++y) c[x] += sh.copies[y][bin];
          sh.hist[0][bin] = c[x];
        } else {
          c[x] = sh.hist[d][bin];
        }
      }
      if (ctas > 1) {
        cluster.sync();
        for (uint32_t q = 1; q < ctas; ++q) {
          const uint4 v = *reinterpret_cast<const uint4*>(&cluster.map_shared_rank(&sh, (part + q) % ctas)->hist[d][kEvictOwn * tid]);
          c[0] += v.x; c[1] += v.y; c[2] += v.z; c[3] += v.w;
        }
      }
      // keys in the bins above: all minus those in the bins up to here
      uint32_t total, upto = 0;
#pragma unroll
      for (uint32_t x = 0; x < kEvictOwn; ++x) upto += c[x];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= uint32_t(o)) upto += x;
      }
      const uint32_t before = warps_before(__shfl_sync(0xffffffffu, upto, 31), sh.warp_count[d & 1], &total);
      uint32_t above = total - before - upto;
#pragma unroll
      for (int x = kEvictOwn - 1; x >= 0; --x) {
        if (above < need && above + c[x] >= need) { sh.bin = kEvictOwn * tid + x; sh.need = need - above; }
        above += c[x];
      }
      __syncthreads();
      prefix |= sh.bin << shift;
      need = sh.need;
    }
    // ---- keys above `prefix` stay, and the first `need` slots of those equal to it ----------------------------------------
    auto key_at = [&](uint32_t i) { return i >= hi ? 0u : (cached ? key_s[i - c_lo] : key_of(i)); };
    auto from_peers = [&](uint32_t EvictShared::*what, uint32_t* all) {
      uint32_t sum = 0, mine = 0;
      for (uint32_t q = 0; q < ctas; ++q) {
        const uint32_t v = ctas > 1 ? cluster.map_shared_rank(&sh, q)->*what : sh.*what;
        if (q < part) mine += v;
        sum += v;
      }
      *all = sum;
      return mine;
    };
    // In one pass over the warp's slots: ties, and the keys above `prefix`, below the budget and not.  The ties that stay are the
    // first ones, and the slots below the budget come first, so both kinds of kept slots follow from the counts.
    uint32_t ties = 0, ties_low = 0, above_low = 0, above_high = 0, total, all;
    for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
      const uint32_t k = key_at(i0 + lane);
      const bool in = i0 + lane < hi;
      const uint32_t eq = __ballot_sync(0xffffffffu, in && k == prefix), gt = __ballot_sync(0xffffffffu, in && k > prefix);
      const uint32_t low = i0 >= p.budget ? 0u : (p.budget - i0 >= 32 ? 0xffffffffu : (1u << (p.budget - i0)) - 1u);
      ties += __popc(eq);
      ties_low += __popc(eq & low);
      above_low += __popc(gt & low);
      above_high += __popc(gt & ~low);
    }
    uint32_t ties_before = warps_before(ties, sh.warp_count[1], &total);
    if (tid == 0) sh.ties = total;
    if (ctas > 1) cluster.sync(); else __syncthreads();
    ties_before += from_peers(&EvictShared::ties, &all);
    const uint32_t ties_kept = need > ties_before ? min(need - ties_before, ties) : 0u, ties_kept_low = min(ties_kept, ties_low);
    const uint32_t low_slots = min(hi, p.budget) - min(lo, p.budget);
    uint32_t total_h, total_m, moved;
    uint32_t hole_at = warps_before(low_slots - above_low - ties_kept_low, sh.warp_count[0], &total_h);
    uint32_t move_at = warps_before(above_high + ties_kept - ties_kept_low, sh.warp_count[1], &total_m);
    if (tid == 0) { sh.holes = total_h; sh.movers = total_m; }
    if (ctas > 1) cluster.sync(); else __syncthreads();
    hole_at += from_peers(&EvictShared::holes, &all);
    move_at += from_peers(&EvictShared::movers, &moved);      // = the holes: as many slots stay as there are below the budget
    int32_t* movers = pos_out + p.budget;                      // until the end of the call the tails of the outputs hold the lists
    int32_t* holes = reinterpret_cast<int32_t*>(mass_out + p.budget);
    uint32_t t = ties_before;
    constexpr int B = 4;                                       // groups of 32 slots under way
    for (uint32_t g0 = lo; g0 < hi; g0 += 32 * B) {
      float m[B];
      int32_t ps[B];
#pragma unroll
      for (int x = 0; x < B; ++x) {
        const uint32_t i = g0 + x * 32 + lane;
        if (i < hi && i < p.budget) {
          m[x] = mass[i];
          ps[x] = pos ? pos[i] : int32_t(i);
        }
      }
#pragma unroll
      for (int x = 0; x < B; ++x) {
        const uint32_t i = g0 + x * 32 + lane, k = key_at(i);
        const bool in = i < hi, low = i < p.budget;
        const uint32_t eq = __ballot_sync(0xffffffffu, in && k == prefix);
        const bool keep = in && (k > prefix || (k == prefix && t + __popc(eq & below) < need));
        t += __popc(eq);
        const uint32_t hb = __ballot_sync(0xffffffffu, in && !keep && low), mb = __ballot_sync(0xffffffffu, keep && !low);
        if (in && !keep && low) holes[hole_at + __popc(hb & below)] = int32_t(i);
        if (keep && !low) movers[move_at + __popc(mb & below)] = int32_t(i);
        if (keep && low) {
          src[i] = int32_t(i);
          mass_out[i] = m[x];
          pos_out[i] = ps[x];
        }
        hole_at += __popc(hb);
        move_at += __popc(mb);
      }
    }
    if (ctas > 1) cluster.sync(); else __syncthreads();       // the lists are complete
    for (uint32_t i = part * kEvictThreads + tid; i < moved; i += ctas * kEvictThreads) {
      const int32_t to = holes[i], from = movers[i];
      src[to] = from;
      mass_out[to] = mass[from];
      pos_out[to] = pos ? pos[from] : from;
    }
    if constexpr (MOVES) {
      constexpr int N = 8;
      const EvictRows r(p, row);
      const uint32_t stride = ctas * kEvictWarps;
      for (uint32_t i = part * kEvictWarps + warp; i < moved; i += N * stride) {
        const uint32_t mine = i + (lane % N) * stride;
        const int hole = mine < moved ? holes[mine] : -1, mover = mine < moved ? movers[mine] : 0;
        int to[N], from[N];
#pragma unroll
        for (int x = 0; x < N; ++x) {
          to[x] = __shfl_sync(0xffffffffu, hole, x);
          from[x] = __shfl_sync(0xffffffffu, mover, x);
        }
        move_slots(p, r, to, from, lane);
      }
    }
  } else {
    for (uint32_t i = part * kEvictThreads + tid; i < len; i += ctas * kEvictThreads) {
      src[i] = int32_t(i);
      mass_out[i] = mass[i];
      pos_out[i] = pos ? pos[i] : int32_t(i);
    }
  }
  if (ctas > 1) cluster.sync(); else __syncthreads();         // the lists have been read (and no CTA leaves while a peer reads its counts)
  for (uint32_t i = kept + part * kEvictThreads + tid; i < p.budget; i += ctas * kEvictThreads) src[i] = -1;
  for (uint32_t i = kept + part * kEvictThreads + tid; i < p.cap; i += ctas * kEvictThreads) { mass_out[i] = 0.f; pos_out[i] = -1; }
}

}  // namespace kuiops

using namespace kuiops;

extern "C" {

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
  if (a.cap > 0x7fffff00u || uint64_t(n) * h_kv * kEvictMaxCluster >= (1ull << 31) || uint64_t(e > ev ? e : ev) * 4 >= (1ull << 31)) return KUIOPS_ELIMIT;
  auto whole = [&](const void* t, uint32_t f, int64_t sn, int64_t sh, int64_t sl) {
    const int64_t v = 16 / elem_bytes;
    return aligned16(t) && f % v == 0 && (n == 1 || sn % v == 0) && (h_kv == 1 || sh % v == 0) && sl % v == 0;
  };
  a.wide = whole(a.K, e, a.k_sn, a.k_sh, a.k_ss) && whole(a.V, ev, a.v_sn, a.v_sh, a.v_ss);
  // A cluster as large as fills the SMs, as long as a CTA has 4096 slots of its own: below that its steps are all latency.
  const uint32_t rows = n * h_kv;
  uint32_t ctas = 1;
  while (ctas < kEvictMaxCluster && rows * ctas < uint32_t(num_sms()) && a.cap > 4096 * ctas) ctas *= 2;
  const uint32_t slice = ((a.cap + ctas - 1) / ctas + 31) & ~31u;
  a.cached = slice <= kEvictMaxKeys ? slice : 0;
  const size_t smem = sizeof(EvictShared) + size_t(a.cached) * 4;
  // A second launch costs some 3 us; the clusters' own warps reach the rate of a few SMs.  (One sequence, 1111 to 1024 slots:
  // 15.5 us a call in one launch, 17.9 in two; 512 rows, 16384 to 8192 slots: 702 us in one, 524 in two.)
  const uint64_t pairs = uint64_t(rows) * (a.budget < a.cap - a.budget ? a.budget : a.cap - a.budget);
  const bool spread = pairs * (e + ev) * elem_bytes > (16u << 20);
  auto kern = spread ? kv_evict_kernel<false> : kv_evict_kernel<true>;
  static std::atomic<uint64_t> configured[2];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KUIOPS_ELAUNCH;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured[spread].load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(EvictShared) + kEvictMaxKeys * 4)) != cudaSuccess)
      return KUIOPS_ELAUNCH;
    configured[spread].fetch_or(bit, std::memory_order_release);
  }
  const uint32_t chunks = (a.budget + 255) / 256;
  if (spread && uint64_t(rows) * chunks >= (1ull << 31)) return KUIOPS_ELIMIT;
  cudaStream_t st = as_stream(stream);
  const int rc = ctas == 1 ? launch_pdl(kern, dim3(rows), dim3(kEvictThreads), smem, st, a, 1u)
                           : launch_cluster_pdl(kern, dim3(rows * ctas), dim3(kEvictThreads), smem, st, ctas, a, ctas);
  if (rc != KUIOPS_OK || !spread) return rc;
  return launch_pdl(kv_evict_move_kernel, dim3(rows * chunks), dim3(256), 0, st, a, chunks);
}

}  // extern "C"
