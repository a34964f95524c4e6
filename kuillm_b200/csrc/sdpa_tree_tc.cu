// Attention of drafted tokens over a KV cache on tcgen05 (16-bit types, up to 128 features per head).
//
// Bound by reading the cache from HBM: every K / V byte is used once per KV head for the G l rows that share it.  A CTA
// owns up to 128 query rows of one (batch, KV head) - G heads x lt drafted positions, one TMA box - and a slice of the
// 64-key tiles: the cache's tiles first, then those of the drafted keys.  K and V tiles arrive through one in-order TMA
// ring (K0 V0 K1 V1 ...); S = Q K^T goes to TMEM (double buffered), the softmax is online with one thread per row, P returns to
// TMEM over the scores it came from and is the A operand of O += P V.  Two CTAs share an SM.
//
// Few rows leave most of the 128 lanes idle, and the softmax of a tile is then one warp's work.  With at most 64 (32) rows
// Q is loaded REP = 2 (4) times, one copy per half (quarter) of the lanes, and each copy takes its own half (quarter) of a
// tile's columns, its P being zero in the others.  A copy keeps its own maximum, sum and O; they are joined at the end like key
// slices.  The products cost the same (their M is 128 in any case).
//
// Masked keys take no part: cache rows behind the key count are zeroed in the V tile before the product, and so are the
// drafted rows' elements that are not finite; those are added at the end to the rows that do see them.
#include "tree.cuh"
#include "tc_ptx.cuh"
#include <type_traits>

namespace kuiops {

constexpr int RTN = 64;                    // keys per tile
constexpr int kTreeThreads = 192;          // warp 0: TMA, warp 1: UMMA issue, warps 2-5: softmax and epilogue
constexpr uint32_t kTreeTmemCols = 256;    // two score buffers at columns 0 and 64, O at column 128
constexpr float kTreeRescale = 8.0f;       // log2 units: O is rescaled when a row's maximum grew by more than 2^8

template <int DD> struct TreeTile {
  static constexpr uint32_t kHalves = DD / 64;
  static constexpr uint32_t kQBytes = 128 * 128 * kHalves;
  static constexpr uint32_t kTBytes = RTN * 128 * kHalves;      // one K or V tile
  static constexpr uint32_t kRing = DD == 128 ? 5 : 9;
  static constexpr uint32_t kSmem = kQBytes + kRing * kTBytes + 256;
  static constexpr uint32_t kStage = DD + 4;                    // floats per staged output row
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs per SM");
  static_assert(128 * kStage * 4 + 2048 <= kRing * kTBytes, "the ring holds the staged rows at the end");
};

struct TreeTcParams {
  TreeArgs a;
  uint32_t G, lt, rows, row_tiles, splits, min_tiles;
  float scale_log2;
  float* partials;
  unsigned int* err;
};

__device__ __forceinline__ uint64_t tree_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = tree_ns();
  while (!tc::mbar_try_wait(bar, parity)) {
    if (tree_ns() - t0 > 2000000000ull) return false;
  }
  return true;
}
// The same for a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool tree_wait_warp(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tree_wait(bar, parity)); }
__device__ __forceinline__ void tree_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// (a0, a1) = (a0, a1) * s + c as one packed instruction
__device__ __forceinline__ void tree_fma2(float& a0, float& a1, float s, float c) {
  asm("{.reg .b64 ra, rb, rc;\n mov.b64 ra, {%0, %1};\n mov.b64 rb, {%2, %2};\n mov.b64 rc, {%3, %3};\n"
      " fma.rn.f32x2 ra, ra, rb, rc;\n mov.b64 {%0, %1}, ra;}"
      : "+f"(a0), "+f"(a1) : "f"(s), "f"(c));
}
__device__ __forceinline__ void tree_add2(float& a0, float& a1, float b0, float b1) {
  asm("{.reg .b64 ra, rb;\n mov.b64 ra, {%0, %1};\n mov.b64 rb, {%2, %3};\n add.rn.f32x2 ra, ra, rb;\n mov.b64 {%0, %1}, ra;}"
      : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
// Bits of a 16-bit element that are all set in infinities and NaN alone.
template <typename T> __device__ __forceinline__ uint32_t exponent_bits() { return std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u; }

template <typename T, int DD, int REP>
__global__ void __launch_bounds__(kTreeThreads, 2)
sdpa_tree_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmKd, const __grid_constant__ CUtensorMap tmVd, const TreeTcParams p) {
  using TT = TreeTile<DD>;
  constexpr uint32_t R = TT::kRing;
  constexpr uint32_t SPAN = 128 / REP;                 // lanes of one copy of the rows
  constexpr int NC = RTN / REP;                        // columns of a tile that a copy takes
  // the 128-byte swizzle needs a 1024-byte aligned base; two CTAs leave no room to pad, so a misaligned one is reported
  extern __shared__ __align__(1024) unsigned char smem[];
  if ((tc::smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0u, 40u);
    return;
  }
  unsigned char* q_s = smem;
  unsigned char* ring = q_s + TT::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + R * TT::kTBytes);
  uint64_t* q_full = bars;               // 1
  uint64_t* t_full = bars + 1;           // R: tile landed
  uint64_t* t_empty = t_full + R;        // R: the products that read the tile have completed
  uint64_t* s_full = t_empty + R;        // 2
  uint64_t* p_ready = s_full + 2;        // 1
  uint64_t* o_done = p_ready + 1;        // 1
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 1);
  int* odd_flag = reinterpret_cast<int*>(tmem_slot + 1);      // a drafted value was not finite
  static_assert((1 + 2 * R + 4) * 8 + 8 <= 256, "barriers");

  const TreeArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // row tiles of the same keys are neighbours in the grid: the second one finds the tiles in L2
  uint32_t u = blockIdx.x;
  const uint32_t rt = u % p.row_tiles; u /= p.row_tiles;
  const uint32_t split = u % p.splits; u /= p.splits;
  const uint32_t kvh = u % a.h_kv, b = u / a.h_kv;
  const uint32_t l0 = rt * p.lt;

  if (threadIdx.x == 0) {
    tc::prefetch_tmap(&tmQ); tc::prefetch_tmap(&tmK); tc::prefetch_tmap(&tmV); tc::prefetch_tmap(&tmKd); tc::prefetch_tmap(&tmVd);
    tc::mbar_init(q_full, 1);
    for (uint32_t i = 0; i < R; ++i) { tc::mbar_init(&t_full[i], 1); tc::mbar_init(&t_empty[i], 1); }
    tc::mbar_init(&s_full[0], 1);
    tc::mbar_init(&s_full[1], 1);
    tc::mbar_init(p_ready, 4);
    tc::mbar_init(o_done, 1);
    *odd_flag = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, kTreeTmemCols);
    tc::tmem_relinquish();
  }
  if (p.rows < SPAN) {
    // rows of the tile that no copy fills must not feed stale bit patterns into the product
    const uint32_t per = (SPAN - p.rows) * 8;          // 16-byte pieces per copy and half
    for (uint32_t i = threadIdx.x; i < per * REP * TT::kHalves; i += kTreeThreads) {
      const uint32_t blk = i / per, o = i % per, copy = blk % REP, half = blk / REP;
      *reinterpret_cast<int4*>(q_s + half * (128 * 128) + (copy * SPAN + p.rows) * 128 + o * 16) = make_int4(0, 0, 0, 0);
    }
    tc::fence_proxy_async();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_S = tmem_base, tmem_O = tmem_base + 128;
  pdl_wait();          // every operand may still be being written by earlier kernels
  pdl_trigger();

  const uint32_t S = a.kv_lens ? clamp_len(a.kv_lens[b], a.s) : a.s;
  const uint32_t cache_tiles = (S + RTN - 1) / RTN, tiles = cache_tiles + (a.l + RTN - 1) / RTN;
  const uint32_t per = max((tiles + p.splits - 1) / p.splits, p.min_tiles);
  const uint32_t t_lo = min(split * per, tiles), t_hi = min(t_lo + per, tiles), n_tiles = t_hi - t_lo;

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------------------
    if (lane == 0 && n_tiles > 0) {
      tc::mbar_expect_tx(q_full, REP * TT::kHalves * p.rows * 128u);
#pragma unroll
      for (uint32_t half = 0; half < TT::kHalves; ++half)
#pragma unroll
        for (uint32_t c = 0; c < REP; ++c)
          tc::tma_load_4d(q_s + half * (128 * 128) + c * SPAN * 128, &tmQ, q_full, int(half * 64), int(l0), int(kvh * p.G), int(b));
      uint32_t n = 0;
      for (; n < 2 * n_tiles; ++n) {
        const uint32_t buf = n % R, ph = (n / R) & 1, t = t_lo + (n >> 1);
        if (n >= R && !tree_wait(&t_empty[buf], ph ^ 1)) { atomicCAS(p.err, 0u, 41u); break; }
        unsigned char* dst = ring + buf * TT::kTBytes;
        const bool drafted = t >= cache_tiles;
        const CUtensorMap* tm = drafted ? ((n & 1) ? &tmVd : &tmKd) : ((n & 1) ? &tmV : &tmK);
        const int key0 = int((drafted ? t - cache_tiles : t) * RTN);
        tc::mbar_expect_tx(&t_full[buf], TT::kTBytes);
#pragma unroll
        for (uint32_t half = 0; half < TT::kHalves; ++half)
          tc::tma_load_4d(dst + half * (RTN * 128), tm, &t_full[buf], int(half * 64), key0, int(kvh), int(b));
      }
      if (n < 2 * n_tiles) {               // gave up: the copies in flight must land before the CTA leaves
        for (uint32_t m = n > R ? n - R : 0; m < n; ++m) tree_wait(&t_full[m % R], (m / R) & 1);
        tree_wait(q_full, 0);
      }
    }
  } else if (warp == 1) {
    // ------------------------------ UMMA issuer -------------------------------------------
    if (lane == 0 && n_tiles > 0) {
      constexpr int is_bf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      constexpr uint32_t idesc_qk = tc::make_idesc(is_bf16, 0, 0, 128, RTN);
      constexpr uint32_t idesc_pv = tc::make_idesc(is_bf16, 0, 1, 128, DD);
      bool ok = tree_wait(q_full, 0);
      if (!ok) atomicCAS(p.err, 0u, 42u);
      // a descriptor's low bits are the address in 16-byte units: tiles and steps are additions
      const uint64_t q_desc = tc::make_smem_desc(tc::smem_u32(q_s), 16, 1024), k_desc0 = tc::make_smem_desc(tc::smem_u32(ring), 16, 1024);
      const uint64_t v_desc0 = tc::make_smem_desc(tc::smem_u32(ring), RTN * 128, 1024);
      auto issue_qk = [&](uint32_t j) -> bool {
        const uint32_t n = 2 * j, buf = n % R;
        const uint64_t k_desc = k_desc0 + buf * (TT::kTBytes >> 4);
        if (!tree_wait(&t_full[buf], (n / R) & 1)) { atomicCAS(p.err, 0u, 43u); return false; }
        tc::tc_fence_after();
#pragma unroll
        for (uint32_t hh = 0; hh < TT::kHalves; ++hh)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc::umma_f16(tmem_S + (j & 1) * RTN, q_desc + (hh * (128 * 128) + kk * 32) / 16, k_desc + (hh * (RTN * 128) + kk * 32) / 16, idesc_qk,
                         (hh | kk) ? 1u : 0u);
        tc::umma_commit(&t_empty[buf]);
        tc::umma_commit(&s_full[j & 1]);
        return true;
      };
      if (ok) ok = issue_qk(0);
      for (uint32_t j = 0; j < n_tiles && ok; ++j) {
        const uint32_t n = 2 * j + 1, buf = n % R;
        const uint64_t v_desc = v_desc0 + buf * (TT::kTBytes >> 4);
        // The next tile's scores are computed during this tile's softmax.  Their buffer holds P of tile j - 1, whose
        // product was issued before (the pipe runs in order), and the softmax left it when p_ready of j - 1 arrived.
        if (j + 1 < n_tiles && !issue_qk(j + 1)) { ok = false; break; }
        if (!tree_wait(p_ready, j & 1)) { atomicCAS(p.err, 0u, 44u); ok = false; break; }
        if (!tree_wait(&t_full[buf], (n / R) & 1)) { atomicCAS(p.err, 0u, 45u); ok = false; break; }
        tc::tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          tc::umma_f16_ts(tmem_O, tmem_S + (j & 1) * RTN + kk * 8, v_desc + kk * 128, idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
        tc::umma_commit(&t_empty[buf]);
        tc::umma_commit(o_done);
      }
    }
  } else {
    // ------------------------------ softmax + epilogue ------------------------------------
    const uint32_t quarter = warp & 3;
    const uint32_t r128 = quarter * 32 + lane;            // lane of the tile
    const uint32_t copy = (quarter * 32) / SPAN, r = r128 % SPAN;
    const uint32_t li = l0 + r % p.lt;
    const bool row_valid = r < p.rows && li < a.l;
    const uint32_t lane_addr = (quarter * 32) << 16;
    const uint32_t tid = threadIdx.x - 64;
    const unsigned char* mrow = a.mask + int64_t(b) * a.mask_sn + size_t(row_valid ? li : 0) * a.l;
    float m_used = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (uint32_t j = 0; j < n_tiles && ok; ++j) {
      const uint32_t t = t_lo + j;
      const bool drafted = t >= cache_tiles;
      const uint32_t key0 = (drafted ? t - cache_tiles : t) * RTN;
      const uint32_t nv = min(uint32_t(RTN), (drafted ? a.l : S) - key0);     // keys of the tile
      uint64_t vis = ~0ull;                                                   // this copy's columns the row sees
      if (drafted) {
        vis = 0;
        if (row_valid) {
#pragma unroll 16
          for (int c = 0; c < NC; ++c) {
            const uint32_t k = copy * NC + c;
            if (k < nv && mrow[key0 + k] != 0) vis |= 1ull << c;
          }
        }
      } else if (nv < RTN) {
        const int left = int(nv) - int(copy * NC);
        vis = left <= 0 ? 0ull : (left >= 64 ? ~0ull : (1ull << left) - 1ull);
      }
      if (!tree_wait_warp(&s_full[j & 1], (j >> 1) & 1)) { atomicCAS(p.err, 0u, 46u); ok = false; break; }
      tc::tc_fence_after();
      float sv[NC];
      const uint32_t s_addr = tmem_S + (j & 1) * RTN + lane_addr + copy * NC;
      if constexpr (NC == 64) { tc::tmem_ld32(s_addr, sv); tc::tmem_ld32(s_addr + 32, sv + 32); }
      else if constexpr (NC == 32) tc::tmem_ld32(s_addr, sv);
      else tc::tmem_ld16(s_addr, sv);
      tc::tmem_ld_wait();
      if (drafted || nv < RTN) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (!((vis >> c) & 1ull)) sv[c] = -INFINITY;
        // What lies behind the keys, and drafted elements that are not finite, would reach rows that do not see them
        // through 0 x inf: they leave the V tile before the product.
        const uint32_t n = 2 * j + 1, buf = n % R;
        if (!tree_wait_warp(&t_full[buf], (n / R) & 1)) { atomicCAS(p.err, 0u, 47u); ok = false; break; }
        unsigned char* vt = ring + buf * TT::kTBytes;
        for (uint32_t i = tid; i < RTN * 8 * TT::kHalves; i += 128) {         // 16-byte pieces; rows are 8 of them per half
          const uint32_t key = (i >> 3) % RTN;
          uint4* at = reinterpret_cast<uint4*>(vt) + i;
          if (key >= nv) {
            *at = make_uint4(0, 0, 0, 0);
          } else if (drafted) {
            uint4 w = *at;
            uint32_t* e = reinterpret_cast<uint32_t*>(&w);
            const uint32_t eb = exponent_bits<T>();
            bool odd = false;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if ((e[x] & eb) == eb) { e[x] &= 0xFFFF0000u; odd = true; }
              if (((e[x] >> 16) & eb) == eb) { e[x] &= 0x0000FFFFu; odd = true; }
            }
            if (odd) { *at = w; *odd_flag = 1; }
          }
        }
        tc::fence_proxy_async();
      }
      float mx = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
#pragma unroll
      for (int c = 4; c < NC; c += 4) mx = fmaxf(mx, fmaxf(fmaxf(sv[c], sv[c + 1]), fmaxf(sv[c + 2], sv[c + 3])));
      mx *= p.scale_log2;                       // scale > 0: the maximum commutes with the scaling
      float corr = 1.f;
      if (mx > m_used + kTreeRescale || m_used == -INFINITY) {
        const float m_new = fmaxf(mx, m_used);
        if (m_used != -INFINITY) corr = fast_ex2(m_used - m_new);      // nothing accumulated before the first key
        m_used = m_new;
      }
      const float nmm = (m_used == -INFINITY) ? 0.f : -m_used;
      float r0 = 0.f, r1 = 0.f, r2 = 0.f, r3 = 0.f;
      uint32_t pk[NC / 2];
#pragma unroll
      for (int c = 0; c < NC; c += 4) {
        tree_fma2(sv[c], sv[c + 1], p.scale_log2, nmm);
        tree_fma2(sv[c + 2], sv[c + 3], p.scale_log2, nmm);
        const float e0 = fast_ex2(sv[c]), e1 = fast_ex2(sv[c + 1]), e2 = fast_ex2(sv[c + 2]), e3 = fast_ex2(sv[c + 3]);
        tree_add2(r0, r1, e0, e1);
        tree_add2(r2, r3, e2, e3);
        pk[c / 2] = pack2<T>(e0, e1);
        pk[c / 2 + 1] = pack2<T>(e2, e3);
      }
      l_run = l_run * corr + ((r0 + r1) + (r2 + r3));
      if (j > 0) {
        // waited for in every tile: a parity wait tells a phase from the one before it only
        if (!tree_wait_warp(o_done, (j - 1) & 1)) { atomicCAS(p.err, 0u, 48u); ok = false; break; }
        tc::tc_fence_after();
        if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
          for (int c0 = 0; c0 < DD; c0 += 16) {
            float ov[16];
            tc::tmem_ld16(tmem_O + lane_addr + c0, ov);
            tc::tmem_ld_wait();
            uint32_t ou[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) ou[c] = __float_as_uint(ov[c] * corr);
            tc::tmem_st16(tmem_O + lane_addr + c0, ou);
          }
          tc::tmem_st_wait();
        }
      }
      // P over the scores it came from: column c holds keys 2 c and 2 c + 1, zero outside this copy's columns
      const uint32_t p_addr = tmem_S + (j & 1) * RTN + lane_addr;
      if constexpr (REP == 1) {
        tc::tmem_st32(p_addr, pk);
      } else if constexpr (REP == 2) {
        const uint32_t zero[16] = {};
        tc::tmem_st16(p_addr + copy * 16, pk);
        tc::tmem_st16(p_addr + (copy ^ 1) * 16, zero);
      } else {
        const uint32_t zero[8] = {};
        tmem_st8(p_addr + copy * 8, pk);
#pragma unroll
        for (int x = 1; x < 4; ++x) tmem_st8(p_addr + ((copy + x) & 3) * 8, zero);
      }
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_ready);
    }
    if (ok && n_tiles > 0 && !tree_wait_warp(o_done, (n_tiles - 1) & 1)) { atomicCAS(p.err, 0u, 49u); ok = false; }
    tc::tc_fence_after();
    // every tile has been consumed: the ring becomes the staging area (a wait that ran out leaves it alone)
    float* stage = reinterpret_cast<float*>(ring);
    float2* ml = reinterpret_cast<float2*>(stage + 128 * TT::kStage);        // per lane: maximum, sum
    float2* fin = ml + 128;                                                   // per row: joined maximum, sum
    if (ok) ml[r128] = make_float2(m_used, l_run);
    tree_barrier();
    if (ok) {
      float mm = m_used;
#pragma unroll
      for (int c = 0; c < REP; ++c) mm = fmaxf(mm, ml[c * SPAN + r].x);
      const float f = m_used == -INFINITY ? (l_run == 0.f ? 0.f : 1.f) : (REP == 1 ? 1.f : fast_ex2(m_used - mm));
      if (copy == 0) {
        float den = 0.f;
#pragma unroll
        for (int c = 0; c < REP; ++c) {
          const float2 x = ml[c * SPAN + r];
          den += x.y * (x.x == -INFINITY ? 1.f : (REP == 1 ? 1.f : fast_ex2(x.x - mm)));
        }
        fin[r] = make_float2(mm, den);
      }
#pragma unroll
      for (int c0 = 0; c0 < DD; c0 += 16) {
        float ov[16];
        if (n_tiles > 0) {
          tc::tmem_ld16(tmem_O + lane_addr + c0, ov);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) ov[c] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 16; c += 4)
          *reinterpret_cast<float4*>(stage + r128 * TT::kStage + c0 + c) = make_float4(ov[c] * f, ov[c + 1] * f, ov[c + 2] * f, ov[c + 3] * f);
      }
    }
    tree_barrier();
    if (ok) {
      const uint32_t cols = (a.ev + 3) / 4;
      const bool odd = *odd_flag != 0;
      for (uint32_t i = tid; i < p.rows * cols; i += 128) {
        const uint32_t row = i / cols, c = (i % cols) * 4, pos = l0 + row % p.lt, head = kvh * p.G + row / p.lt;
        if (pos >= a.l) continue;
        float4 o = *reinterpret_cast<const float4*>(stage + row * TT::kStage + c);
#pragma unroll
        for (int k = 1; k < REP; ++k) {
          const float4 x = *reinterpret_cast<const float4*>(stage + (k * SPAN + row) * TT::kStage + c);
          o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        }
        if (odd) {
          // drafted elements that were taken out of the product, for the rows that see them
          const unsigned char* mr = a.mask + int64_t(b) * a.mask_sn + size_t(pos) * a.l;
          const uint32_t d_lo = t_lo > cache_tiles ? (t_lo - cache_tiles) * RTN : 0;
          const uint32_t d_hi = t_hi > cache_tiles ? min((t_hi - cache_tiles) * RTN, a.l) : 0;
          for (uint32_t k = d_lo; k < d_hi; ++k) {
            if (mr[k] == 0) continue;
            const T* v = static_cast<const T*>(a.DV) + int64_t(b) * a.dv_sn + int64_t(kvh) * a.dv_sh + int64_t(k) * a.dv_sl + c;
            const float x0 = ElemTraits<T>::to_f(v[0]), x1 = ElemTraits<T>::to_f(v[1]), x2 = ElemTraits<T>::to_f(v[2]), x3 = ElemTraits<T>::to_f(v[3]);
            if (!isfinite(x0)) o.x += x0;
            if (!isfinite(x1)) o.y += x1;
            if (!isfinite(x2)) o.z += x2;
            if (!isfinite(x3)) o.w += x3;
          }
        }
        const float2 md = fin[row];
        const uint64_t orow = (uint64_t(b) * a.h + head) * a.l + pos;
        if (p.splits == 1) {
          const float inv = md.y == 0.f ? 0.f : 1.f / md.y;
          T* dst = static_cast<T*>(a.out) + int64_t(b) * a.o_sn + int64_t(head) * a.o_sh + int64_t(pos) * a.o_sl + c;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
          if (c == 0 && a.lse) a.lse[orow] = md.y == 0.f ? -INFINITY : (md.x + log2f(md.y)) * 0.6931471805599453f;
        } else {
          float* rec = tree_record(p.partials, orow, p.splits, split, a.ev);
          *reinterpret_cast<float4*>(rec + c) = o;
          if (c == 0) *reinterpret_cast<float2*>(rec + tree_record_floats(a.ev) - 4) = md;
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base, kTreeTmemCols);
  }
}

bool sdpa_tree_tc_eligible(const TreeArgs& a) {
  if (a.dtype != KUIOPS_BF16 && a.dtype != KUIOPS_F16) return false;
  if (!(a.scale > 0.f)) return false;                       // the row maximum is taken before scaling
  if (a.e > 128 || a.ev > 128 || a.e % 8 || a.ev % 8) return false;
  if (a.h / a.h_kv > 128) return false;
  // what a TMA descriptor takes: 16-byte aligned bases and strides
  auto ok = [&](const void* t, int64_t sn, int64_t sh, int64_t sl, uint32_t heads, uint32_t rows) {
    auto st = [](int64_t s) { return s > 0 && s % 8 == 0 && uint64_t(s) * 2 < (1ull << 40); };
    return aligned16(t) && (rows == 1 || st(sl)) && (heads == 1 || st(sh)) && (a.n == 1 || st(sn));
  };
  if (!ok(a.Q, a.q_sn, a.q_sh, a.q_sl, a.h, a.l) || !ok(a.out, a.o_sn, a.o_sh, a.o_sl, a.h, a.l)) return false;
  if (!ok(a.DK, a.dk_sn, a.dk_sh, a.dk_sl, a.h_kv, a.l) || !ok(a.DV, a.dv_sn, a.dv_sh, a.dv_sl, a.h_kv, a.l)) return false;
  return a.s == 0 || (ok(a.K, a.k_sn, a.k_sh, a.k_ss, a.h_kv, a.s) && ok(a.V, a.v_sn, a.v_sh, a.v_ss, a.h_kv, a.s));
}

struct TreeTcPlan { uint32_t lt, rows, row_tiles, splits, min_tiles; };

static TreeTcPlan tree_tc_plan(const TreeArgs& a) {
  TreeTcPlan pl;
  const uint32_t G = a.h / a.h_kv, most = 128 / G;
  pl.row_tiles = (a.l + most - 1) / most;
  pl.lt = (a.l + pl.row_tiles - 1) / pl.row_tiles;
  pl.row_tiles = (a.l + pl.lt - 1) / pl.lt;
  pl.rows = G * pl.lt;
  const uint64_t units = uint64_t(a.n) * a.h_kv * pl.row_tiles, slots = 2ull * num_sms();
  const uint32_t tiles = (a.s + RTN - 1) / RTN + (a.l + RTN - 1) / RTN;
  pl.min_tiles = 2;
  uint64_t splits = slots / units;
  if (splits > tiles / 2) splits = tiles / 2;
  pl.splits = splits < 1 ? 1u : (splits > 64 ? 64u : uint32_t(splits));
  return pl;
}

uint32_t sdpa_tree_tc_splits(const TreeArgs& a) { return tree_tc_plan(a).splits; }

template <typename T, int DD, int REP>
static int tree_tc_launch(const CUtensorMap* m, const TreeTcParams& p, cudaStream_t st) {
  auto kern = sdpa_tree_tc_kernel<T, DD, REP>;
  constexpr size_t smem = TreeTile<DD>::kSmem;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KUIOPS_ELAUNCH;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return KUIOPS_ELAUNCH;
    configured.fetch_or(bit, std::memory_order_release);
  }
  const uint64_t grid = uint64_t(p.a.n) * p.a.h_kv * p.splits * p.row_tiles;
  if (grid >= (1ull << 31)) return KUIOPS_ELIMIT;
  return launch_pdl(kern, dim3(unsigned(grid)), dim3(kTreeThreads), smem, st, m[0], m[1], m[2], m[3], m[4], p);
}

template <typename T, int DD>
static int tree_tc_launch_rep(const CUtensorMap* m, const TreeTcParams& p, cudaStream_t st) {
  if (p.rows <= 32) return tree_tc_launch<T, DD, 4>(m, p, st);
  if (p.rows <= 64) return tree_tc_launch<T, DD, 2>(m, p, st);
  return tree_tc_launch<T, DD, 1>(m, p, st);
}

int sdpa_tree_tc(const TreeArgs& a, float* partials, cudaStream_t st) {
  const TreeTcPlan pl = tree_tc_plan(a);
  TreeTcParams p = {};
  p.a = a; p.G = a.h / a.h_kv; p.lt = pl.lt; p.rows = pl.rows; p.row_tiles = pl.row_tiles; p.splits = pl.splits; p.min_tiles = pl.min_tiles;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.partials = partials;
  p.err = tc_error_word_device();
  if (!p.err) return KUIOPS_ELAUNCH;
  CUtensorMap m[5];
  auto enc = [&](CUtensorMap* t, const void* base, uint32_t feat, uint32_t rows, uint32_t heads, int64_t sn, int64_t sh, int64_t sl,
                 uint32_t box_rows, uint32_t box_heads) {
    // a dimension of extent 1 may carry any stride: give it a legal one
    const uint64_t r = rows > 1 ? uint64_t(sl) : uint64_t(feat + 7) / 8 * 8;
    const uint64_t h = heads > 1 ? uint64_t(sh) : r * rows;
    const uint64_t dims[4] = {feat, rows, heads, a.n};
    const uint64_t strides[4] = {1, r, h, a.n > 1 ? uint64_t(sn) : h * heads};
    const uint32_t box[4] = {64, box_rows, box_heads, 1};
    return encode_tmap_2byte(t, base, 4, dims, strides, box);
  };
  if (!enc(&m[0], a.Q, a.e, a.l, a.h, a.q_sn, a.q_sh, a.q_sl, pl.lt, p.G)) return KUIOPS_EDRIVER;
  if (!enc(&m[3], a.DK, a.e, a.l, a.h_kv, a.dk_sn, a.dk_sh, a.dk_sl, RTN, 1)) return KUIOPS_EDRIVER;
  if (!enc(&m[4], a.DV, a.ev, a.l, a.h_kv, a.dv_sn, a.dv_sh, a.dv_sl, RTN, 1)) return KUIOPS_EDRIVER;
  m[1] = m[3]; m[2] = m[4];                  // an empty cache is never read
  if (a.s > 0) {
    if (!enc(&m[1], a.K, a.e, a.s, a.h_kv, a.k_sn, a.k_sh, a.k_ss, RTN, 1)) return KUIOPS_EDRIVER;
    if (!enc(&m[2], a.V, a.ev, a.s, a.h_kv, a.v_sn, a.v_sh, a.v_ss, RTN, 1)) return KUIOPS_EDRIVER;
  }
  const bool wide = a.e > 64 || a.ev > 64;
  if (a.dtype == KUIOPS_BF16) return wide ? tree_tc_launch_rep<__nv_bfloat16, 128>(m, p, st) : tree_tc_launch_rep<__nv_bfloat16, 64>(m, p, st);
  return wide ? tree_tc_launch_rep<__half, 128>(m, p, st) : tree_tc_launch_rep<__half, 64>(m, p, st);
}

}  // namespace kuiops
