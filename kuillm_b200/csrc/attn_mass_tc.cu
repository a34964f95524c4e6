// Attention weight received per key, on tcgen05 (16-bit types, up to 128 features per head).
//
// Scores are computed transposed, S^T = K Q^T: the 128 lanes of the tile are keys and the columns are query rows (G heads x
// lt positions).  A key's weight is then a sum along one thread's own columns - no exchange between threads, no maximum (the
// rows' log-sum-exp is given), no second product - and what the thread holds at the end is the answer.
//
// One persistent CTA per SM walks (batch, KV head, 128-key tile) items; four groups of four warps (a thread per key) make the
// weights.
//   Up to 64 rows per KV head (decode, a small window): bound by reading K once from HBM.  Four to eight K tiles are in flight,
//   an item is one product, and the groups take items in turn, each with a score buffer of its own, so that a group's
//   latencies (log-sum-exp, scores, the old mass) hide behind three other items.  (8 entries, 8 KV heads, 16001 keys, one
//   token: 50 us, 0.76 of the copy rate; 4 entries of 64 rows a head over up to 8191 keys: 34 us.)
//   More rows (a window, a prompt): bound by the exponentials, 16 per clock and SM, then by the products.  Tiles of 128 rows
//   stream past a resident K tile (128 columns: a 64-column product would be bound by shared memory, whose A operand it reads
//   twice as often) and every group takes 32 columns of each.  Items are dealt in alternating direction, which evens out a causal mask's
//   falling work per item.  (Making a quarter of the exponentials by a polynomial in the FMA pipe was slower, 396 against
//   361 us for an 8192-token prompt, which now takes 323 us at 1965 MHz: the instructions it takes are what the scheduler has least of.)
//
// Weights and their sums stay in 32 bits.  Beside its score a weight is off by the special-function unit's 2^-22 and by the rounding of
// lse to the log2 domain, 2^-24 |lse|.
#include "tree.cuh"
#include "tc_ptx.cuh"
#include <type_traits>

namespace kuiops {

constexpr int kMassGroups = 4;
// warp 0: TMA, warp 1: UMMA issue, warps 2-17: weights, then a warp per 32 columns that prepares the rows' values
template <int NQ> constexpr int kMassRowWarps = NQ < 32 ? 1 : NQ / 32;
template <int NQ> constexpr int kMassThreads = 64 + 128 * kMassGroups + 32 * kMassRowWarps<NQ>;
constexpr uint32_t MKT = 128;              // keys per item
constexpr uint32_t kMassLens = 256;        // key counts kept in shared memory
constexpr uint32_t kMassS = 4;             // score buffers

// NQ columns per tile; 128 = the form that streams row tiles, else all rows are one tile.
template <int DD, int NQ> struct MassTile {
  static constexpr bool kStream = NQ == 128;
  static constexpr uint32_t kHalves = DD / 64;
  static constexpr uint32_t kKBytes = MKT * 128 * kHalves;
  static constexpr uint32_t kQBytes = NQ * 128 * kHalves;
  static constexpr uint32_t kKRing = kStream ? 2 : (DD == 64 ? 8 : (NQ == 64 ? 4 : (NQ == 32 ? 5 : 6)));
  static constexpr uint32_t kQRing = kStream ? 4 : kKRing;
  static constexpr uint32_t kRows = kStream ? 32 : NQ;    // columns of a warp
  static constexpr uint32_t kBars = 2 * (kKRing + 2 * kQRing + kMassS) + 2;
  static constexpr uint32_t kSmem = kKRing * kKBytes + kQRing * kQBytes + kBars * 8 + kMassLens * 4 + kQRing * (2 * NQ + 4) * 4 + (kStream ? 4 * 4 * 128 * 4 : 0);
  static_assert(kSmem <= 227 * 1024, "one CTA per SM");
};

struct MassTcParams {
  MassArgs a;
  uint32_t G, lt, rows, q_tiles, items, n_cols;
  FastDiv by_item, by_heads, by_lens, by_lt;      // adjacent items, KV heads, key counts, positions per row tile
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

// Packed fp32 pairs.
struct F2 { float x, y; };
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("{.reg .b64 ra, rb, rc;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n mov.b64 rc, {%6, %7};\n"
      " fma.rn.f32x2 ra, ra, rb, rc;\n mov.b64 {%0, %1}, ra;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("{.reg .b64 ra, rb;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n add.rn.f32x2 ra, ra, rb;\n mov.b64 {%0, %1}, ra;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ F2 both(float v) { return F2{v, v}; }
// One (batch, KV head, key tile) and the row tiles that can see it.
struct MassItem {
  uint32_t b, kvh, g, key0, len, qt0, qt1;
};

__device__ __forceinline__ bool mass_item(const MassTcParams& p, const uint32_t* lens_s, uint32_t round, MassItem& it) {
  // Round r deals items r * grid .. in ascending or descending CTA order.  With several row tiles the key tiles come first, so
  // that a causal mask's work falls with the item; with one the CTAs of a round read adjacent keys.
  const uint32_t id = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  if (round * gridDim.x >= p.items) return false;
  if (id >= p.items) { it.qt0 = it.qt1 = 0; it.key0 = p.a.s; return true; }      // no item left for this turn
  const uint32_t hi = p.by_item.div(id), lo = id - hi * p.by_item.d;
  const uint32_t kt = p.q_tiles > 1 ? hi : lo, u = p.q_tiles > 1 ? lo : hi;
  it.b = p.by_heads.div(u);
  it.kvh = u - it.b * p.a.h_kv;
  it.g = it.b - p.by_lens.div(it.b) * p.a.lens_n;
  it.key0 = kt * MKT;
  it.len = !p.a.kv_lens ? p.a.s : (it.g < kMassLens ? lens_s[it.g] : clamp_len(p.a.kv_lens[it.g], p.a.s));
  it.qt0 = 0;
  it.qt1 = it.key0 < it.len ? p.q_tiles : 0;
  if (p.q_tiles > 1 && p.a.is_causal && !p.a.q_lens) {
    // position i sees key0 when i >= key0 - (len - l)
    const int64_t first = int64_t(it.key0) - (int64_t(it.len) - int64_t(p.a.l));
    if (first > 0) it.qt0 = min(p.by_lt.div(uint32_t(first)), it.qt1);
  }
  return true;
}

template <typename T, int DD, int NQ>
__global__ void __launch_bounds__(kMassThreads<NQ>, 1)
attn_mass_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const MassTcParams p) {
  using MT = MassTile<DD, NQ>;
  constexpr bool STREAM = MT::kStream;
  constexpr uint32_t KR = MT::kKRing, QR = MT::kQRing;
  constexpr uint32_t TMEM = kMassS * NQ;
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
  uint64_t* r_full = q_empty + QR;       // QR: log-sum-exp and limits of a tile's rows
  uint64_t* r_empty = r_full + QR;
  uint64_t* s_full = r_empty + QR;       // kMassS
  uint64_t* s_empty = s_full + kMassS;   // kMassS
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_empty + kMassS);
  uint32_t* lens_s = reinterpret_cast<uint32_t*>(bars + MT::kBars);
  constexpr uint32_t RS = 2 * NQ + 4;    // words of a stage: -lse (log2 domain), limits, the least limit of each 32 rows
  float* row_s = reinterpret_cast<float*>(lens_s + kMassLens);
  float* part_s = row_s + QR * RS;       // [4][group][128] sums of the groups, for four items
  const MassArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tc::prefetch_tmap(&tmQ); tc::prefetch_tmap(&tmK);
    for (uint32_t i = 0; i < KR; ++i) { tc::mbar_init(&k_full[i], 1); tc::mbar_init(&k_empty[i], 1); }
    for (uint32_t i = 0; i < QR; ++i) {
      tc::mbar_init(&q_full[i], 1); tc::mbar_init(&q_empty[i], 1);
      tc::mbar_init(&r_full[i], kMassRowWarps<NQ>); tc::mbar_init(&r_empty[i], STREAM ? 4 * kMassGroups : 4);
    }
    // scores: the product's completion, and the issuer's word that the rows' values are there
    for (uint32_t i = 0; i < kMassS; ++i) { tc::mbar_init(&s_full[i], 2); tc::mbar_init(&s_empty[i], STREAM ? 4 * kMassGroups : 4); }
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, TMEM);
    tc::tmem_relinquish();
  }
  if (p.rows < NQ) {
    // rows of the tile that TMA does not fill feed columns nobody counts, but no stale bit patterns either
    const uint32_t per = (NQ - p.rows) * 8;
    for (uint32_t i = threadIdx.x; i < per * QR * MT::kHalves; i += kMassThreads<NQ>) {
      const uint32_t blk = i / per, o = i % per;         // blk = stage * halves + half
      *reinterpret_cast<int4*>(q_s + blk * (NQ * 128) + p.rows * 128 + o * 16) = make_int4(0, 0, 0, 0);
    }
    tc::fence_proxy_async();
  }
  pdl_wait();
  if (a.kv_lens)
    for (uint32_t i = threadIdx.x; i < min(a.lens_n, kMassLens); i += kMassThreads<NQ>) lens_s[i] = clamp_len(a.kv_lens[i], a.s);
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
            tc::tma_load_4d(q_s + qb * MT::kQBytes + half * (NQ * 128), &tmQ, &q_full[qb], int(half * 64), int(qt * p.lt), int(it.kvh * p.G), int(it.b));
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
      // a descriptor's low bits are the address in 16-byte units: stages and steps are additions
      const uint64_t k_desc0 = tc::make_smem_desc(tc::smem_u32(k_s), 16, 1024), q_desc0 = tc::make_smem_desc(tc::smem_u32(q_s), 16, 1024);
      uint32_t nk = 0, nq = 0;
      bool ok = true;
      for (uint32_t round = 0; ok && mass_item(p, lens_s, round, it); ++round) {
        if (it.qt0 >= it.qt1) continue;
        const uint32_t kb = nk % KR;
        const uint64_t k_desc = k_desc0 + kb * (MT::kKBytes >> 4);
        if (!mass_wait(&k_full[kb], (nk / KR) & 1)) { atomicCAS(p.err, 0u, 53u); break; }
        for (uint32_t qt = it.qt0; qt < it.qt1; ++qt, ++nq) {
          const uint32_t qb = nq % QR, sb = nq % kMassS;
          const uint64_t q_desc = q_desc0 + qb * (MT::kQBytes >> 4);
          if (!mass_wait(&q_full[qb], (nq / QR) & 1)) { atomicCAS(p.err, 0u, 54u); ok = false; break; }
          if (nq >= kMassS && !mass_wait(&s_empty[sb], ((nq / kMassS) & 1) ^ 1)) { atomicCAS(p.err, 0u, 55u); ok = false; break; }
          tc::tc_fence_after();
#pragma unroll
          for (uint32_t hh = 0; hh < MT::kHalves; ++hh)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc::umma_f16(tmem_base + sb * NQ, k_desc + (hh * (MKT * 128) + kk * 32) / 16, q_desc + (hh * (NQ * 128) + kk * 32) / 16, idesc,
                           (hh | kk) ? 1u : 0u);
          tc::umma_commit(&q_empty[qb]);
          tc::umma_commit(&s_full[sb]);
          // one wait of this thread in place of one of every weight warp
          if (!mass_wait(&r_full[qb], (nq / QR) & 1)) { atomicCAS(p.err, 0u, 58u); ok = false; break; }
          tc::mbar_arrive(&s_full[sb]);
        }
        tc::umma_commit(&k_empty[kb]);
        ++nk;
      }
    }
  } else if (warp >= 2 + 4 * kMassGroups) {
    // ------------------------------ the rows' values: -lse and key limit, two tiles ahead -------
    const uint32_t w = warp - (2 + 4 * kMassGroups), row = w * 32 + lane, gh = row / p.lt, ri = row - gh * p.lt;
    const bool row_in = row < p.rows;
    uint32_t round = 0, qt = 0;
    bool more = true;
    it.qt0 = it.qt1 = 0;
    const float* lse_row = a.lse;
    const int64_t* lim_row = a.q_lens;
    struct Ahead { float lse; long long lim; uint32_t len; bool valid; };
    auto fetch = [&]() {
      Ahead f{0.f, 0, 0, false};
      while (more && qt >= it.qt1) {
        more = mass_item(p, lens_s, round++, it);
        qt = it.qt0;
        if (more && qt < it.qt1) {
          lse_row = a.lse + (size_t(it.b) * a.h + it.kvh * p.G + gh) * a.l;
          if (a.q_lens) lim_row = a.q_lens + size_t(it.g) * a.l;
        }
      }
      if (!more) return f;
      const uint32_t li = qt++ * p.lt + ri;
      f.valid = true;
      f.len = it.len;
      if (row_in && li < a.l) {
        f.lse = lse_row[li];
        f.lim = a.q_lens ? lim_row[li] : (a.is_causal ? (long long)li + 1 + (long long)it.len - (long long)a.l : (long long)it.len);
      }
      return f;
    };
    Ahead f0 = fetch(), f1 = fetch();
    for (uint32_t nq = 0; f0.valid; ++nq) {
      const Ahead f2 = fetch();
      const uint32_t qb = nq % QR;
      if (nq >= QR && !__all_sync(0xffffffffu, mass_wait(&r_empty[qb], ((nq / QR) & 1) ^ 1))) { atomicCAS(p.err, 0u, 57u); break; }
      float* rs = row_s + qb * RS;
      float nl = -1.4426950408889634f * f0.lse;
      uint32_t lim = clamp_len(f0.lim, f0.len);
      if (isinf(nl)) { nl = 0.f; lim = 0; }                  // saw nothing, or is not to be counted
      if (row < NQ) {
        rs[row] = nl;
        reinterpret_cast<uint32_t*>(rs)[NQ + row] = lim;
      }
      const uint32_t low = __reduce_min_sync(0xffffffffu, row < NQ ? lim : 0xffffffffu);
      if (lane == 0) reinterpret_cast<uint32_t*>(rs)[2 * NQ + w] = low;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&r_full[qb]);
      f0 = f1;
      f1 = f2;
    }
  } else {
    // ------------------------------ weights: one key per thread ---------------------------
    constexpr uint32_t W = MT::kRows;                     // columns of this warp
    constexpr uint32_t C = W < 32 ? W : 32;               // columns at a time
    const uint32_t quarter = warp & 3, key = quarter * 32 + lane, group = uint32_t(warp - 2) >> 2;
    const uint32_t col0 = STREAM ? group * 32 : 0;
    const uint32_t s_base = tmem_base + ((quarter * 32) << 16) + col0;
    bool ok = true;
    uint32_t tile = 0, n_item = 0;
    for (uint32_t round = 0; mass_item(p, lens_s, round, it); ++round) {
      const uint32_t j = it.key0 + key;
      const bool any = it.qt0 < it.qt1;
      // without row tiles a round is dealt by its number, with one by the tile's: a group waits for every use of its score buffer
      // in turn
      if (!STREAM && (any ? tile++ : round) % kMassGroups != group) continue;
      const size_t o = (size_t(it.b) * a.h_kv + it.kvh) * a.s + j;
      float total = 0.f, old = 0.f;
      // the group that writes the item: with row tiles the one whose turn it is among those, else the one the round falls to
      const bool writes = !STREAM || (any ? n_item : round) % kMassGroups == group;
      if (writes && a.mass && j < a.s) old = a.mass[o];
      uint32_t nq = STREAM ? tile : tile - 1;
      for (uint32_t qt = it.qt0; qt < it.qt1; ++qt, ++nq) {
        const uint32_t sb = nq % kMassS, qb = nq % QR;
        if (ok && !__all_sync(0xffffffffu, mass_wait(&s_full[sb], (nq / kMassS) & 1))) {
          atomicCAS(p.err, 0u, 56u);
          ok = false;
        }
        tc::tc_fence_after();
        const float* rs = row_s + qb * RS;
        float part = 0.f;
#pragma unroll
        for (uint32_t h = 0; h < W / C; ++h) {
          float sv[C];
          if constexpr (C == 16) tc::tmem_ld16(s_base + sb * NQ, sv);
          else tc::tmem_ld32(s_base + sb * NQ + h * C, sv);
          tc::tmem_ld_wait();
          if (h == W / C - 1) {
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s_empty[sb]);
          }
          const float* nlc = rs + col0 + h * C;
          const uint32_t* lmc = reinterpret_cast<const uint32_t*>(rs) + NQ + col0 + h * C;
          if (reinterpret_cast<const uint32_t*>(rs)[2 * NQ + (col0 + h * C) / 32] >= it.key0 + MKT) {
            // every row counts for every key of the tile
            F2 r0 = both(0.f), r1 = both(0.f);
#pragma unroll
            for (uint32_t c = 0; c < C; c += 4) {
              const float4 x = *reinterpret_cast<const float4*>(nlc + c);
              const F2 u = fma2(F2{sv[c], sv[c + 1]}, both(p.scale_log2), F2{x.x, x.y});
              const F2 v = fma2(F2{sv[c + 2], sv[c + 3]}, both(p.scale_log2), F2{x.z, x.w});
              r0 = add2(r0, F2{fast_ex2(u.x), fast_ex2(u.y)});
              r1 = add2(r1, F2{fast_ex2(v.x), fast_ex2(v.y)});
            }
            r0 = add2(r0, r1);
            part += r0.x + r0.y;
          } else {
#pragma unroll
            for (uint32_t c = 0; c < C; ++c) {
              const float w = fast_ex2(fmaf(sv[c], p.scale_log2, nlc[c]));
              part += j < lmc[c] ? w : 0.f;
            }
          }
        }
        total += part;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&r_empty[qb]);
      }
      if constexpr (STREAM) {
        if (any) {
          // The groups' sums meet in shared memory, in group order.  Only the group whose turn it is waits for the others; they go
          // on with the next item.  A buffer comes up again four items later, and before that every group has waited for all the
          // others once, in an item that the reader of this one had to reach first.
          tile = nq;
          const uint32_t slot = n_item++ % kMassGroups;
          float* part = part_s + slot * (kMassGroups * 128) + key;
          part[group * 128] = total;
          if (writes) {
            asm volatile("bar.sync %0, 512;" ::"r"(1 + slot) : "memory");
            total = (part[0] + part[128]) + (part[256] + part[384]);
          } else {
            asm volatile("bar.arrive %0, 512;" ::"r"(1 + slot) : "memory");
          }
        }
      }
      if (writes && j < a.s && (a.mass != a.out || j < it.len)) a.out[o] = old + (j < it.len ? total : 0.f);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base, TMEM);
  }
}

bool attn_mass_tc_eligible(const MassArgs& a) {
  if (a.dtype != KUIOPS_BF16 && a.dtype != KUIOPS_F16) return false;
  if (a.e > 128 || a.e % 8 || a.h / a.h_kv > 128) return false;
  if (uint64_t(a.n) * a.h_kv * ((a.s + MKT - 1) / MKT) >= (1ull << 31)) return false;
  auto ok = [&](const void* t, int64_t sn, int64_t sh, int64_t sl, uint32_t heads, uint32_t rows) {
    auto st = [](int64_t s) { return s > 0 && s % 8 == 0 && uint64_t(s) * 2 < (1ull << 40); };
    return aligned16(t) && (rows == 1 || st(sl)) && (heads == 1 || st(sh)) && (a.n == 1 || st(sn));
  };
  return ok(a.Q, a.q_sn, a.q_sh, a.q_sl, a.h, a.l) && ok(a.K, a.k_sn, a.k_sh, a.k_ss, a.h_kv, a.s);
}

template <typename T, int DD, int NQ>
static int mass_tc_launch(const CUtensorMap& mq, const CUtensorMap& mk, const MassTcParams& p, cudaStream_t st) {
  auto kern = attn_mass_tc_kernel<T, DD, NQ>;
  constexpr size_t smem = MassTile<DD, NQ>::kSmem;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KUIOPS_ELAUNCH;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return KUIOPS_ELAUNCH;
    configured.fetch_or(bit, std::memory_order_release);
  }
  const uint32_t slots = uint32_t(num_sms());
  return launch_pdl(kern, dim3(p.items < slots ? p.items : slots), dim3(kMassThreads<NQ>), smem, st, mq, mk, p);
}

template <typename T, int DD>
static int mass_tc_launch_rows(const CUtensorMap& mq, const CUtensorMap& mk, const MassTcParams& p, uint32_t nq, cudaStream_t st) {
  if (nq == 16) return mass_tc_launch<T, DD, 16>(mq, mk, p, st);
  if (nq == 32) return mass_tc_launch<T, DD, 32>(mq, mk, p, st);
  if (nq == 64) return mass_tc_launch<T, DD, 64>(mq, mk, p, st);
  return mass_tc_launch<T, DD, 128>(mq, mk, p, st);
}

int attn_mass_tc(const MassArgs& a, cudaStream_t st) {
  MassTcParams p = {};
  p.a = a; p.G = a.h / a.h_kv;
  const uint64_t all = uint64_t(p.G) * a.l;
  const uint32_t nq = all <= 16 ? 16 : (all <= 32 ? 32 : (all <= 64 ? 64 : 128));
  // as few row tiles as hold all rows, of even size
  p.q_tiles = (a.l + nq / p.G - 1) / (nq / p.G);
  p.lt = (a.l + p.q_tiles - 1) / p.q_tiles;
  p.q_tiles = (a.l + p.lt - 1) / p.lt;
  p.rows = p.G * p.lt;
  p.n_cols = (p.rows + 15) & ~15u;
  const uint32_t units = a.n * a.h_kv, key_tiles = (a.s + MKT - 1) / MKT;
  p.items = units * key_tiles;
  p.by_item.set(p.q_tiles > 1 ? units : key_tiles);
  p.by_heads.set(a.h_kv);
  p.by_lens.set(a.lens_n);
  p.by_lt.set(p.lt);
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
    return a.e > 64 ? mass_tc_launch_rows<__nv_bfloat16, 128>(mq, mk, p, nq, st) : mass_tc_launch_rows<__nv_bfloat16, 64>(mq, mk, p, nq, st);
  return a.e > 64 ? mass_tc_launch_rows<__half, 128>(mq, mk, p, nq, st) : mass_tc_launch_rows<__half, 64>(mq, mk, p, nq, st);
}

}  // namespace kuiops
