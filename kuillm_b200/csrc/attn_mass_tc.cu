// Attention weight received per key, on tcgen05 (16-bit types, up to 128 features per head).
//
// Scores are computed transposed, S^T = K Q^T: the 128 lanes of the tile are keys and the columns are query rows (G heads x
// lt positions, at most 64).  A key's weight is then a sum along one thread's own columns - no exchange between threads, no
// maximum (the rows' log-sum-exp is given), no second product - and what the thread holds at the end is the answer.
//
// For a few rows the kernel is bound by reading K once from HBM: persistent CTAs, two to an SM, walk (batch, KV head,
// 128-key tile) items and keep two K tiles in flight each.  For many rows it is bound by the exponentials (16 per clock and SM): the
// rows' tiles stream past a resident K tile, four score buffers in TMEM keep the products ahead.  Items are dealt in
// alternating direction, which evens out a causal mask's falling work per tile.
#include "tree.cuh"
#include "tc_ptx.cuh"
#include <type_traits>

namespace kuiops {

// warp 0: TMA, warp 1: UMMA issue, then one group of four warps per 32 columns (one key per thread): two groups give the
// wide tiles' exponentials four warps per scheduler to hide latencies with (one group of 64 columns: 588 us for the 8192-token
// prompt, two: see below)
template <int NQ> constexpr int kMassGroups = NQ == 64 ? 2 : 1;
template <int NQ> constexpr int kMassThreads = 64 + 128 * kMassGroups<NQ>;
constexpr uint32_t MKT = 128;              // keys per item
constexpr uint32_t MQR = 64;               // query rows per tile, at most
constexpr uint32_t kMassLens = 256;        // key counts kept in shared memory

template <int DD> struct MassTile {
  static constexpr uint32_t kHalves = DD / 64;
  static constexpr uint32_t kKBytes = MKT * 128 * kHalves;
  static constexpr uint32_t kQBytes = MQR * 128 * kHalves;
  static constexpr uint32_t kKRing = DD == 128 ? 2 : 4;
  static constexpr uint32_t kQRing = DD == 128 ? 2 : 4;
  static constexpr uint32_t kBars = 1 + 2 * (kKRing + kQRing) + 8;
  static constexpr uint32_t kSmem = kKRing * kKBytes + kQRing * kQBytes + kBars * 8 + 16 + kMassLens * 4 + 8 * 64 * 8 + 2 * 128 * 4;
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs per SM");
};
constexpr uint32_t kMassS = 4;             // score buffers of 64 columns

struct MassTcParams {
  MassArgs a;
  uint32_t G, lt, rows, q_tiles, key_tiles, units, n_cols;
  float scale_log2;
  unsigned int* err;
};

__device__ __forceinline__ bool mass_wait(uint64_t* bar, uint32_t parity) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  while (!tc::mbar_try_wait(bar, parity)) {
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > 2000000000ull) return false;
  }
  return true;
}

// (a0, a1) = (a0, a1) * s + (c0, c1) and (a0, a1) += (b0, b1) as packed instructions
__device__ __forceinline__ void mass_fma2(float& a0, float& a1, float s, float c0, float c1) {
  asm("{.reg .b64 ra, rb, rc;\n mov.b64 ra, {%0, %1};\n mov.b64 rb, {%2, %2};\n mov.b64 rc, {%3, %4};\n"
      " fma.rn.f32x2 ra, ra, rb, rc;\n mov.b64 {%0, %1}, ra;}"
      : "+f"(a0), "+f"(a1) : "f"(s), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mass_add2(float& a0, float& a1, float b0, float b1) {
  asm("{.reg .b64 ra, rb;\n mov.b64 ra, {%0, %1};\n mov.b64 rb, {%2, %3};\n add.rn.f32x2 ra, ra, rb;\n mov.b64 {%0, %1}, ra;}"
      : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}

// One (batch, KV head, key tile) and the row tiles that can see it.
struct MassItem {
  uint32_t b, kvh, g, key0, len, qt0, qt1;
};

__device__ __forceinline__ bool mass_item(const MassTcParams& p, const uint32_t* lens_s, uint32_t round, MassItem& it) {
  // round r deals items r * grid .. in ascending or descending CTA order; key tiles ascend, so the work falls
  const uint64_t id = uint64_t(round) * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  if (id >= uint64_t(p.units) * p.key_tiles) return false;
  const uint32_t kt = uint32_t(id / p.units), u = uint32_t(id % p.units);
  it.b = u / p.a.h_kv; it.kvh = u % p.a.h_kv; it.g = it.b % p.a.lens_n;
  it.key0 = kt * MKT;
  it.len = !p.a.kv_lens ? p.a.s : (it.g < kMassLens ? lens_s[it.g] : clamp_len(p.a.kv_lens[it.g], p.a.s));
  it.qt0 = 0;
  it.qt1 = it.key0 < it.len ? p.q_tiles : 0;
  if (p.a.is_causal && !p.a.q_lens) {
    // position i sees key0 when i >= key0 - (len - l)
    const int64_t first = int64_t(it.key0) - (int64_t(it.len) - int64_t(p.a.l));
    if (first > 0) it.qt0 = min(uint32_t(first) / p.lt, it.qt1);
  }
  return true;
}

template <typename T, int DD, int NQ>
__global__ void __launch_bounds__(kMassThreads<NQ>, 2)
attn_mass_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const MassTcParams p) {
  using MT = MassTile<DD>;
  constexpr uint32_t KR = MT::kKRing, QR = MT::kQRing;
  constexpr int GROUPS = kMassGroups<NQ>, THREADS = kMassThreads<NQ>;
  extern __shared__ __align__(1024) unsigned char smem[];
  if ((tc::smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0u, 50u);
    return;
  }
  unsigned char* k_s = smem;
  unsigned char* q_s = k_s + KR * MT::kKBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(q_s + QR * MT::kQBytes);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + KR;
  uint64_t* q_full = k_empty + KR;
  uint64_t* q_empty = q_full + QR;
  uint64_t* s_full = q_empty + QR;       // kMassS
  uint64_t* s_empty = s_full + kMassS;   // kMassS
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_empty + kMassS);
  uint32_t* lens_s = tmem_slot + 4;
  float* row_s = reinterpret_cast<float*>(lens_s + kMassLens);            // per warp [2][32] -lse (log2 domain) and [2][32] limits
  float* part_s = row_s + 8 * 128;                                         // [2][128] sums of the second group
  const MassArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tc::prefetch_tmap(&tmQ); tc::prefetch_tmap(&tmK);
    for (uint32_t i = 0; i < KR; ++i) { tc::mbar_init(&k_full[i], 1); tc::mbar_init(&k_empty[i], 1); }
    for (uint32_t i = 0; i < QR; ++i) { tc::mbar_init(&q_full[i], 1); tc::mbar_init(&q_empty[i], 1); }
    for (uint32_t i = 0; i < kMassS; ++i) { tc::mbar_init(&s_full[i], 1); tc::mbar_init(&s_empty[i], 4 * GROUPS); }
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, kMassS * MQR);
    tc::tmem_relinquish();
  }
  if (p.rows < NQ) {
    // rows of the tile that TMA does not fill feed columns nobody reads, but no stale bit patterns either
    const uint32_t per = (NQ - p.rows) * 8;
    for (uint32_t i = threadIdx.x; i < per * QR * MT::kHalves; i += THREADS) {
      const uint32_t blk = i / per, o = i % per;         // blk = stage * halves + half
      *reinterpret_cast<int4*>(q_s + blk * (MQR * 128) + p.rows * 128 + o * 16) = make_int4(0, 0, 0, 0);
    }
    tc::fence_proxy_async();
  }
  pdl_wait();
  if (a.kv_lens)
    for (uint32_t i = threadIdx.x; i < min(a.lens_n, kMassLens); i += THREADS) lens_s[i] = clamp_len(a.kv_lens[i], a.s);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();

  MassItem it;
  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------------------
    if (lane == 0) {
      uint32_t nk = 0, nq = 0;
      bool ok = true;
      for (uint32_t round = 0; ok && mass_item(p, lens_s, round, it); ++round) {
        if (it.qt0 >= it.qt1) continue;
        const uint32_t kb = nk % KR;
        if (nk >= KR && !mass_wait(&k_empty[kb], ((nk / KR) & 1) ^ 1)) { atomicCAS(p.err, 0u, 51u); break; }
        tc::mbar_expect_tx(&k_full[kb], MT::kKBytes);
#pragma unroll
        for (uint32_t half = 0; half < MT::kHalves; ++half)
          tc::tma_load_4d(k_s + kb * MT::kKBytes + half * (MKT * 128), &tmK, &k_full[kb], int(half * 64), int(it.key0), int(it.kvh), int(it.b));
        ++nk;
        for (uint32_t qt = it.qt0; qt < it.qt1; ++qt, ++nq) {
          const uint32_t qb = nq % QR;
          if (nq >= QR && !mass_wait(&q_empty[qb], ((nq / QR) & 1) ^ 1)) { atomicCAS(p.err, 0u, 52u); ok = false; break; }
          tc::mbar_expect_tx(&q_full[qb], MT::kHalves * p.rows * 128u);
#pragma unroll
          for (uint32_t half = 0; half < MT::kHalves; ++half)
            tc::tma_load_4d(q_s + qb * MT::kQBytes + half * (MQR * 128), &tmQ, &q_full[qb], int(half * 64), int(qt * p.lt), int(it.kvh * p.G), int(it.b));
        }
      }
      // the copies in flight must land before the CTA leaves (they have, unless a wait ran out)
      for (uint32_t m = nk > KR ? nk - KR : 0; m < nk; ++m) mass_wait(&k_full[m % KR], (m / KR) & 1);
      for (uint32_t m = nq > QR ? nq - QR : 0; m < nq; ++m) mass_wait(&q_full[m % QR], (m / QR) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------ UMMA issuer -------------------------------------------
    if (lane == 0) {
      constexpr int is_bf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      const uint32_t idesc = tc::make_idesc(is_bf16, 0, 0, MKT, int(p.n_cols));
      uint32_t nk = 0, nq = 0;
      bool ok = true;
      for (uint32_t round = 0; ok && mass_item(p, lens_s, round, it); ++round) {
        if (it.qt0 >= it.qt1) continue;
        const uint32_t kb = nk % KR, ka = tc::smem_u32(k_s + kb * MT::kKBytes);
        if (!mass_wait(&k_full[kb], (nk / KR) & 1)) { atomicCAS(p.err, 0u, 53u); break; }
        for (uint32_t qt = it.qt0; qt < it.qt1; ++qt, ++nq) {
          const uint32_t qb = nq % QR, sb = nq % kMassS, qa = tc::smem_u32(q_s + qb * MT::kQBytes);
          if (!mass_wait(&q_full[qb], (nq / QR) & 1)) { atomicCAS(p.err, 0u, 54u); ok = false; break; }
          if (nq >= kMassS && !mass_wait(&s_empty[sb], ((nq / kMassS) & 1) ^ 1)) { atomicCAS(p.err, 0u, 55u); ok = false; break; }
          tc::tc_fence_after();
#pragma unroll
          for (uint32_t hh = 0; hh < MT::kHalves; ++hh)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint64_t da = tc::make_smem_desc(ka + hh * (MKT * 128) + kk * 32, 16, 1024);
              const uint64_t db = tc::make_smem_desc(qa + hh * (MQR * 128) + kk * 32, 16, 1024);
              tc::umma_f16(tmem_base + sb * MQR, da, db, idesc, (hh | kk) ? 1u : 0u);
            }
          tc::umma_commit(&q_empty[qb]);
          tc::umma_commit(&s_full[sb]);
        }
        tc::umma_commit(&k_empty[kb]);
        ++nk;
      }
    }
  } else {
    // ------------------------------ weights: one key per thread ---------------------------
    const uint32_t quarter = warp & 3, key = quarter * 32 + lane, group = uint32_t(warp - 2) >> 2;
    constexpr int W = NQ < 32 ? NQ : 32;                  // columns of this warp: group * 32 ..
    const uint32_t s_base = tmem_base + ((quarter * 32) << 16) + group * 32;
    float* nl_s = row_s + (warp - 2) * 128;
    uint32_t* lim_s = reinterpret_cast<uint32_t*>(nl_s + 64);
    const uint32_t row = group * 32 + lane, gh = row / p.lt, ri = row % p.lt;      // the row this lane looks after
    const bool row_in = row < p.rows;
    uint32_t nq = 0, n_item = 0;
    bool ok = true;
    for (uint32_t round = 0; mass_item(p, lens_s, round, it); ++round) {
      const uint32_t j = it.key0 + key;
      float total = 0.f;
      // -lse and limit of the lane's row, one tile ahead
      float nl = 0.f;
      uint32_t lim = 0;
      const float* lse_row = a.lse + (size_t(it.b) * a.h + it.kvh * p.G + gh) * a.l;
      auto fetch = [&](uint32_t qt) {
        const uint32_t li = qt * p.lt + ri;
        nl = 0.f; lim = 0;
        if (row_in && qt < it.qt1 && li < a.l) {
          nl = -1.4426950408889634f * lse_row[li];
          if (a.q_lens) lim = clamp_len(a.q_lens[size_t(it.g) * a.l + li], it.len);
          else if (a.is_causal) lim = clamp_len((long long)li + 1 + (long long)it.len - (long long)a.l, it.len);
          else lim = it.len;
        }
      };
      fetch(it.qt0);
      for (uint32_t qt = it.qt0; qt < it.qt1; ++qt, ++nq) {
        const uint32_t buf = (nq & 1) * 32, sb = nq % kMassS;
        if (isinf(nl)) { nl = 0.f; lim = 0; }             // saw nothing, or is not to be counted
        nl_s[buf + lane] = nl;
        lim_s[buf + lane] = lim;
        const bool all = __all_sync(0xffffffffu, lim >= it.key0 + MKT);      // every row counts for every key of the tile
        fetch(qt + 1);
        if (ok && !__all_sync(0xffffffffu, mass_wait(&s_full[sb], (nq / kMassS) & 1))) { atomicCAS(p.err, 0u, 56u); ok = false; }
        tc::tc_fence_after();
        float sv[W];
        if constexpr (W == 16) tc::tmem_ld16(s_base + sb * MQR, sv);
        else tc::tmem_ld32(s_base + sb * MQR, sv);
        tc::tmem_ld_wait();
        tc::tc_fence_before();
        __syncwarp();                                      // the row's values are in place, too
        if (lane == 0) tc::mbar_arrive(&s_empty[sb]);
        float r0 = 0.f, r1 = 0.f, r2 = 0.f, r3 = 0.f;
        if (all) {
#pragma unroll
          for (int c = 0; c < W; c += 4) {
            const float4 x = *reinterpret_cast<const float4*>(nl_s + buf + c);
            mass_fma2(sv[c], sv[c + 1], p.scale_log2, x.x, x.y);
            mass_fma2(sv[c + 2], sv[c + 3], p.scale_log2, x.z, x.w);
            mass_add2(r0, r1, fast_ex2(sv[c]), fast_ex2(sv[c + 1]));
            mass_add2(r2, r3, fast_ex2(sv[c + 2]), fast_ex2(sv[c + 3]));
          }
        } else {
#pragma unroll
          for (int c = 0; c < W; ++c) {
            const float w = fast_ex2(fmaf(sv[c], p.scale_log2, nl_s[buf + c]));
            r0 += j < lim_s[buf + c] ? w : 0.f;
          }
        }
        total += (r0 + r1) + (r2 + r3);
      }
      if constexpr (GROUPS == 2) {
        // the second group's sums come through shared memory; two buffers and one meeting per item: a thread that is an item
        // ahead writes the other buffer
        float* part = part_s + (n_item++ & 1) * 128;
        if (group == 1) part[key] = total;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (group == 0) total += part[key];
      }
      if (group == 0 && j < a.s) {
        const size_t o = (size_t(it.b) * a.h_kv + it.kvh) * a.s + j;
        if (a.mass != a.out || j < it.len) a.out[o] = (a.mass ? a.mass[o] : 0.f) + (j < it.len ? total : 0.f);
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base, kMassS * MQR);
  }
}

bool attn_mass_tc_eligible(const MassArgs& a) {
  if (a.dtype != KUIOPS_BF16 && a.dtype != KUIOPS_F16) return false;
  if (a.e > 128 || a.e % 8 || a.h / a.h_kv > MQR) return false;
  auto ok = [&](const void* t, int64_t sn, int64_t sh, int64_t sl, uint32_t heads, uint32_t rows) {
    auto st = [](int64_t s) { return s > 0 && s % 8 == 0 && uint64_t(s) * 2 < (1ull << 40); };
    return aligned16(t) && (rows == 1 || st(sl)) && (heads == 1 || st(sh)) && (a.n == 1 || st(sn));
  };
  return ok(a.Q, a.q_sn, a.q_sh, a.q_sl, a.h, a.l) && ok(a.K, a.k_sn, a.k_sh, a.k_ss, a.h_kv, a.s);
}

template <typename T, int DD, int NQ>
static int mass_tc_launch(const CUtensorMap& mq, const CUtensorMap& mk, const MassTcParams& p, cudaStream_t st) {
  auto kern = attn_mass_tc_kernel<T, DD, NQ>;
  constexpr size_t smem = MassTile<DD>::kSmem;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KUIOPS_ELAUNCH;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return KUIOPS_ELAUNCH;
    configured.fetch_or(bit, std::memory_order_release);
  }
  const uint64_t items = uint64_t(p.units) * p.key_tiles, slots = 2ull * num_sms();
  return launch_pdl(kern, dim3(unsigned(items < slots ? items : slots)), dim3(kMassThreads<NQ>), smem, st, mq, mk, p);
}

template <typename T, int DD>
static int mass_tc_launch_rows(const CUtensorMap& mq, const CUtensorMap& mk, MassTcParams& p, cudaStream_t st) {
  p.n_cols = (p.rows + 15) & ~15u;
  if (p.rows <= 16) return mass_tc_launch<T, DD, 16>(mq, mk, p, st);
  if (p.rows <= 32) return mass_tc_launch<T, DD, 32>(mq, mk, p, st);
  return mass_tc_launch<T, DD, 64>(mq, mk, p, st);
}

int attn_mass_tc(const MassArgs& a, cudaStream_t st) {
  MassTcParams p = {};
  p.a = a; p.G = a.h / a.h_kv;
  // as few row tiles as hold all rows, of even size
  p.q_tiles = (a.l + MQR / p.G - 1) / (MQR / p.G);
  p.lt = (a.l + p.q_tiles - 1) / p.q_tiles;
  p.q_tiles = (a.l + p.lt - 1) / p.lt;
  p.rows = p.G * p.lt;
  p.key_tiles = (a.s + MKT - 1) / MKT;
  const uint64_t units = uint64_t(a.n) * a.h_kv;
  if (units >= (1ull << 31)) return KUIOPS_ELIMIT;
  p.units = uint32_t(units);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.err = tc_error_word_device();
  if (!p.err) return KUIOPS_ELAUNCH;
  CUtensorMap mq, mk;
  auto enc = [&](CUtensorMap* t, const void* base, uint32_t rows, uint32_t heads, int64_t sn, int64_t sh, int64_t sl, uint32_t box_rows, uint32_t box_heads) {
    // a dimension of extent 1 may carry any stride: give it a legal one
    const uint64_t r = rows > 1 ? uint64_t(sl) : uint64_t(a.e);
    const uint64_t h = heads > 1 ? uint64_t(sh) : r * rows;
    const uint64_t dims[4] = {a.e, rows, heads, a.n};
    const uint64_t strides[4] = {1, r, h, a.n > 1 ? uint64_t(sn) : h * heads};
    const uint32_t box[4] = {64, box_rows, box_heads, 1};
    return encode_tmap_2byte(t, base, 4, dims, strides, box);
  };
  if (!enc(&mq, a.Q, a.l, a.h, a.q_sn, a.q_sh, a.q_sl, p.lt, p.G)) return KUIOPS_EDRIVER;
  if (!enc(&mk, a.K, a.s, a.h_kv, a.k_sn, a.k_sh, a.k_ss, MKT, 1)) return KUIOPS_EDRIVER;
  if (a.dtype == KUIOPS_BF16)
    return a.e > 64 ? mass_tc_launch_rows<__nv_bfloat16, 128>(mq, mk, p, st) : mass_tc_launch_rows<__nv_bfloat16, 64>(mq, mk, p, st);
  return a.e > 64 ? mass_tc_launch_rows<__half, 128>(mq, mk, p, st) : mass_tc_launch_rows<__half, 64>(mq, mk, p, st);
}

}  // namespace kuiops
