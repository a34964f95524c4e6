// Attention of drafted tokens over a KV cache on tcgen05 (16-bit types, up to 128 features per head).
//
// Bound by reading the cache from HBM: every K / V byte is used once per KV head for the G l rows that share it.  The tiles of 64
// keys of every unit (batch entry, KV head) - the cache's first, then the drafted ones - form one list, and every CTA takes an
// equal range of it, so that ragged key counts leave no SM idle; a range covers one or more segments (consecutive tiles of a unit).
// A segment that is a whole unit writes its rows; the others leave records, which a second kernel joins.  (Joining them in the CTA
// that finishes a unit last was slower, 87 against 69 us for 16 x 27 rows over 4096 keys: four warps cannot hide it.)  Rows beyond 128
// per unit (G heads x lt drafted positions, one TMA box) go to further CTAs with the same range, which find the tiles in L2.
// 32 / 8 heads of 128, replayed at 1965 MHz: 16 sequences x 27 rows over 2000 to 4001 keys 64 us (the stream alone 39 us, 5 TB/s); 2 x 64 rows
// over 65000 keys 171 us, where no unit is busy for more than a third of the time (counted over 16000 keys: tensor 28 %, special functions
// 29 %, L2 24 %, DRAM 30 %) and each tile's chain from scores to product is what is waited for; 8 rows over 517 keys 12.7 us, the set-up of two launches.
//
// K and V tiles arrive through one in-order TMA ring (K0 V0 K1 V1 ...); S = Q K^T goes to TMEM (double buffered), the softmax
// is online with one thread per row, P returns to TMEM over the scores it came from and is the A operand of O += P V.  Two
// CTAs share an SM.
//
// Few rows leave most of the 128 lanes idle, and the softmax of a tile is then one warp's work.  With at most 64 (32) rows
// Q is loaded REP = 2 (4) times, one copy per half (quarter) of the lanes, and each copy takes its own half (quarter) of a
// tile's columns, its P being zero in the others.  A copy keeps its own maximum, sum and O; they are joined at the end like key
// slices.  The products cost the same (their M is 128 in any case).
//
// Masked keys take no part: cache rows behind the key count are zeroed in the V tile before the product, and so are the
// drafted rows' elements that are not finite; those are added at the end to the rows that do see them.  The cache's own values
// go into the product as they are, where an infinity among them meets the zeros of the other copies (and weights that round to
// zero) and comes out as NaN: a segment whose O is not finite throughout reads its values again and puts such elements right
// (odd_patch).  A finite cache pays one multiply-add per element of O for the question.
#include "tree.cuh"
#include "tc_ptx.cuh"
#include <type_traits>

namespace kuiops {

constexpr int RTN = 64;                    // keys per tile
constexpr int kTreeThreads = 192;          // warp 0: TMA, warp 1: UMMA issue, warps 2-5: softmax and epilogue
constexpr uint32_t kTreeTmemCols = 256;    // two score buffers at columns 0 and 64, O at column 128
constexpr float kTreeRescale = 8.0f;       // log2 units: O is rescaled when a row's maximum grew by more than 2^8

template <int DD, int REP> struct TreeTile {
  static constexpr uint32_t kHalves = DD / 64;
  static constexpr uint32_t kQBytes = 128 * 128 * kHalves;
  static constexpr uint32_t kTBytes = RTN * 128 * kHalves;      // one K or V tile
  // copies of the rows are joined through a staging area of 16 columns (rows of 20 words: no bank conflicts)
  static constexpr uint32_t kStage = REP == 1 ? 0 : 128 * 20 * 4 + 128 * 8;
  static constexpr uint32_t kRing = DD == 128 ? (REP == 1 ? 5 : 4) : (REP == 1 ? 9 : 8);
  static constexpr uint32_t kSmem = kQBytes + kRing * kTBytes + kStage + 256;
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs per SM");
};

struct TreeTcParams {
  TreeArgs a;
  uint32_t G, lt, rows, row_tiles, ranges, min_places;
  float scale_log2;
  float* partials;
  unsigned int* err;
};

// What a segment costs beside its tiles (Q, the mask, the rows' way out), in tiles: the list of tiles that the ranges divide has
// this many empty places ahead of each unit.
constexpr uint32_t kTreeLead = 3;

// (From L2: the joining kernel reads the counts before it waits for the kernel ahead of it.)
__device__ __forceinline__ uint32_t tree_keys(const TreeArgs& a, uint32_t b) {
  return a.kv_lens ? clamp_len(__ldcg(reinterpret_cast<const long long*>(a.kv_lens) + b), a.s) : a.s;
}
__device__ __forceinline__ uint32_t tree_tiles(const TreeArgs& a, uint32_t keys) { return (keys + RTN - 1) / RTN + (a.l + RTN - 1) / RTN; }
// Places of a KV head in all entries and in those before `b` (fewer than 2^31 in all: checked on the host); the whole warp
// takes part.
struct TreePlaces { uint32_t all, before; };
__device__ __forceinline__ TreePlaces tree_places(const TreeArgs& a, uint32_t b) {
  uint32_t all = 0, before = 0;
  for (uint32_t i = threadIdx.x & 31; i < a.n; i += 32) {
    const uint32_t t = tree_tiles(a, tree_keys(a, i)) + kTreeLead;
    all += t;
    if (i < b) before += t;
  }
  return TreePlaces{__reduce_add_sync(0xffffffffu, all), __reduce_add_sync(0xffffffffu, before)};
}
// Record of one output row in range `range`: kind 1 holds the beginning of a unit, kind 0 what continues one.
__device__ __forceinline__ float* tree_tc_record(float* partials, uint32_t ev, uint32_t rows, uint32_t row_tiles, uint32_t range, uint32_t kind,
                                                 uint32_t rt, uint32_t row) {
  return partials + (((uint64_t(range) * 2 + kind) * row_tiles + rt) * rows + row) * tree_record_floats(ev);
}

// Walks the segments of a range.
struct TreeWalk {
  uint32_t pos, end;          // in the list of all places
  uint32_t b, kvh, keys, tiles;   // the unit at pos
  uint32_t v0;                // pos within it
  // the segment taken last: its unit, cache keys, tiles first .. first + count - 1 of `of`
  uint32_t sb, skvh, skeys, first, count, of;
  // The unit that holds place `lo`; the whole warp takes part.
  __device__ void start(const TreeTcParams& p, uint32_t lo, uint32_t hi) {
    pos = lo; end = hi;
    const uint32_t lane = threadIdx.x & 31;
    uint32_t base = 0;
    b = 0; kvh = 0; v0 = 0; keys = 0; tiles = 1;
    if (lo >= hi) return;
    for (uint32_t i0 = 0; i0 < p.a.n; i0 += 32) {
      const uint32_t k = i0 + lane < p.a.n ? tree_keys(p.a, i0 + lane) : 0;
      const uint32_t t = i0 + lane < p.a.n ? tree_tiles(p.a, k) + kTreeLead : 0;
      uint32_t sum = t * p.a.h_kv;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= uint32_t(o)) sum += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, base + sum > lo);
      if (past) {
        const int at = __ffs(past) - 1;
        const uint32_t places = __shfl_sync(0xffffffffu, t, at);
        const uint32_t in = lo - (base + __shfl_sync(0xffffffffu, sum, at) - places * p.a.h_kv);
        keys = __shfl_sync(0xffffffffu, k, at);
        tiles = places - kTreeLead;
        b = i0 + at;
        kvh = in / places;
        v0 = in - kvh * places;
        return;
      }
      base += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  __device__ bool next(const TreeTcParams& p) {
    while (pos < end) {
      const uint32_t places = tiles + kTreeLead, v1 = min(v0 + (end - pos), places);
      sb = b; skvh = kvh; skeys = keys; of = tiles;
      first = v0 > kTreeLead ? v0 - kTreeLead : 0;
      count = (v1 > kTreeLead ? v1 - kTreeLead : 0) - first;
      pos += v1 - v0;
      v0 = v1;
      if (v0 == places && pos < end) {
        v0 = 0;
        if (++kvh == p.a.h_kv) { kvh = 0; keys = tree_keys(p.a, ++b); tiles = tree_tiles(p.a, keys); }
      }
      if (count > 0) return true;
    }
    return false;
  }
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
// The same, and whether `v` is true in any of the four warps' threads.
__device__ __forceinline__ bool tree_barrier_any(bool v) {
  uint32_t any;
  asm volatile("{.reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;}"
               : "=r"(any) : "r"(uint32_t(v)) : "memory");
  return any != 0;
}
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

// NaN where one of v[0 .. N - 1] is not finite, else 0.
template <int N>
__device__ __forceinline__ float odd_test(const float* v) {
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < N; ++c) t[c & 3] = fmaf(v[c], 0.f, t[c & 3]);
  return (t[0] + t[1]) + (t[2] + t[3]);
}

// A segment's values, and the row of the result (`out`, else its record `rec`) that a thread looks after (`row_on`).
template <typename T> struct OddSegment {
  const T *v, *dv;                      // the segment's cache rows, the drafted rows d_lo .. d_hi - 1
  int64_t v_row, dv_row, mask_sk;
  uint32_t keys, d_lo, d_hi, ev;
  bool row_on;
  const unsigned char* mask;
  T* out;
  float* rec;
};
// Elements of the result that came out not finite although the row's weights are: a sum with positive weights is what the visible
// values that are not finite add up to, an infinity, or NaN where both signs or a NaN meet.  Elements whose values are all finite
// stay.  The whole warp takes part, a lane with 16 bytes of a row of V.  Out of line: hardly ever called.
template <typename T>
__device__ __noinline__ void odd_patch(const OddSegment<T> g) {
  const uint32_t lane = threadIdx.x & 31, piece = lane & 3, eb = exponent_bits<T>();
  for (uint32_t c0 = 0; c0 < g.ev; c0 += 32) {
    uint32_t pos = 0, neg = 0, nan = 0;                  // a bit per column
    if (c0 + piece * 8 < g.ev) {
      const T* at = g.v + c0 + piece * 8;
      for (uint32_t k = lane >> 2; k < g.keys; k += 8) {
        const uint4 w = *reinterpret_cast<const uint4*>(at + int64_t(k) * g.v_row);
        const uint32_t e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t y = (e[x / 2] >> (x % 2 * 16)) & 0xFFFFu, bit = 1u << (piece * 8 + x);
          if ((y & eb) != eb) continue;
          if (y & 0x7FFFu & ~eb) nan |= bit;
          else if (y & 0x8000u) neg |= bit;
          else pos |= bit;
        }
      }
    }
    pos = __reduce_or_sync(0xffffffffu, pos);
    neg = __reduce_or_sync(0xffffffffu, neg);
    nan = __reduce_or_sync(0xffffffffu, nan);
    for (uint32_t c = 0; c < 32 && c0 + c < g.ev && g.row_on; ++c) {
      if (isfinite(g.rec ? g.rec[c0 + c] : ElemTraits<T>::to_f(g.out[c0 + c]))) continue;
      float y = 0.f;
      if ((pos >> c) & 1u) y = INFINITY;
      if ((neg >> c) & 1u) y -= INFINITY;
      if ((nan >> c) & 1u) y = NAN;
      for (uint32_t k = g.d_lo; k < g.d_hi; ++k) {
        const float d = ElemTraits<T>::to_f(g.dv[int64_t(k) * g.dv_row + c0 + c]);
        if (!isfinite(d) && g.mask[int64_t(k) * g.mask_sk] != 0) y += d;
      }
      if (y == 0.f) continue;
      if (g.rec) g.rec[c0 + c] = y;
      else g.out[c0 + c] = ElemTraits<T>::from_f(y);
    }
    __syncwarp();
  }
}

// Six warps fill two of the SM's four register files twice and two once, so two CTAs need room for four warps in each: 128
// registers a thread, which is what the bound for 256 threads says (for 192 it would be 168, and one CTA per SM).
template <typename T, int DD, int REP>
__global__ void __launch_bounds__(256, 2)
sdpa_tree_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmKd, const __grid_constant__ CUtensorMap tmVd, const TreeTcParams p) {
  using TT = TreeTile<DD, REP>;
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
  float* stage = reinterpret_cast<float*>(ring + R * TT::kTBytes);        // [128][20]
  float2* ml = reinterpret_cast<float2*>(stage + 128 * 20);               // per lane: maximum, sum
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + R * TT::kTBytes + TT::kStage);
  uint64_t* q_full = bars;               // 1
  uint64_t* q_empty = bars + 1;          // 1: every product of the segment that reads Q has completed
  uint64_t* t_full = bars + 2;           // R: tile landed
  uint64_t* t_empty = t_full + R;        // R: the products that read the tile have completed
  uint64_t* s_full = t_empty + R;        // 2
  uint64_t* p_ready = s_full + 2;        // 1
  uint64_t* o_done = p_ready + 1;        // 1
  uint64_t* o_free = o_done + 1;         // 1: the segment's O has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 1);
  int* odd_flag = reinterpret_cast<int*>(tmem_slot + 1);      // [2] a drafted value of the segment was not finite
  static_assert((2 + 2 * R + 5) * 8 + 12 <= 256, "barriers");

  const TreeArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // row tiles of the same range are neighbours in the grid: the second one finds the tiles in L2
  const uint32_t rt = blockIdx.x % p.row_tiles, range = blockIdx.x / p.row_tiles;
  const uint32_t l0 = rt * p.lt;

  if (threadIdx.x == 0) {
    tc::prefetch_tmap(&tmQ); tc::prefetch_tmap(&tmK); tc::prefetch_tmap(&tmV); tc::prefetch_tmap(&tmKd); tc::prefetch_tmap(&tmVd);
    tc::mbar_init(q_full, 1);
    tc::mbar_init(q_empty, 1);
    for (uint32_t i = 0; i < R; ++i) { tc::mbar_init(&t_full[i], 1); tc::mbar_init(&t_empty[i], 1); }
    tc::mbar_init(&s_full[0], 1);
    tc::mbar_init(&s_full[1], 1);
    tc::mbar_init(p_ready, 4);
    tc::mbar_init(o_done, 1);
    tc::mbar_init(o_free, 4);
    odd_flag[0] = odd_flag[1] = 0;
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

  TreeWalk seg;
  const uint32_t places = tree_places(a, 0).all * a.h_kv, per = max((places + p.ranges - 1) / p.ranges, p.min_places);
  {
    const uint32_t lo = uint32_t(min(uint64_t(range) * per, uint64_t(places)));
    seg.start(p, lo, min(per, places - lo) + lo);
  }

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------------------
    if (lane == 0) {
      uint32_t n = 0, n_seg = 0;
      bool ok = true;
      for (; ok && seg.next(p); ++n_seg) {
        const uint32_t cache_tiles = seg.of - (a.l + RTN - 1) / RTN;
        // the segment's first tiles go ahead of its Q, whose buffer is free once the last products of the segment before ran
        const uint32_t early = min(2 * seg.count, R - 1);
        for (uint32_t i = 0; i < 2 * seg.count && ok; ++i, ++n) {
          const uint32_t buf = n % R, t = seg.first + (i >> 1);
          if (n >= R && !tree_wait(&t_empty[buf], ((n / R) & 1) ^ 1)) { atomicCAS(p.err, 0u, 41u); ok = false; break; }
          unsigned char* dst = ring + buf * TT::kTBytes;
          const bool drafted = t >= cache_tiles;
          const CUtensorMap* tm = drafted ? ((i & 1) ? &tmVd : &tmKd) : ((i & 1) ? &tmV : &tmK);
          const int key0 = int((drafted ? t - cache_tiles : t) * RTN);
          tc::mbar_expect_tx(&t_full[buf], TT::kTBytes);
#pragma unroll
          for (uint32_t half = 0; half < TT::kHalves; ++half)
            tc::tma_load_4d(dst + half * (RTN * 128), tm, &t_full[buf], int(half * 64), key0, int(seg.skvh), int(seg.sb));
          if (i + 1 == early) {
            if (n_seg > 0 && !tree_wait(q_empty, (n_seg - 1) & 1)) { atomicCAS(p.err, 0u, 60u); ok = false; ++n; break; }
            tc::mbar_expect_tx(q_full, REP * TT::kHalves * p.rows * 128u);
#pragma unroll
            for (uint32_t half = 0; half < TT::kHalves; ++half)
#pragma unroll
              for (uint32_t c = 0; c < REP; ++c)
                tc::tma_load_4d(q_s + half * (128 * 128) + c * SPAN * 128, &tmQ, q_full, int(half * 64), int(l0), int(seg.skvh * p.G), int(seg.sb));
          }
        }
      }
      // the copies in flight must land before the CTA leaves (they have, unless a wait ran out)
      for (uint32_t m = n > R ? n - R : 0; m < n; ++m) tree_wait(&t_full[m % R], (m / R) & 1);
      if (!ok && n_seg > 0) tree_wait(q_full, (n_seg - 1) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------ UMMA issuer -------------------------------------------
    if (lane == 0) {
      constexpr int is_bf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      constexpr uint32_t idesc_qk = tc::make_idesc(is_bf16, 0, 0, 128, RTN);
      constexpr uint32_t idesc_pv = tc::make_idesc(is_bf16, 0, 1, 128, DD);
      // a descriptor's low bits are the address in 16-byte units: tiles and steps are additions
      const uint64_t q_desc = tc::make_smem_desc(tc::smem_u32(q_s), 16, 1024), k_desc0 = tc::make_smem_desc(tc::smem_u32(ring), 16, 1024);
      const uint64_t v_desc0 = tc::make_smem_desc(tc::smem_u32(ring), RTN * 128, 1024);
      // g: tiles of this CTA, counted over its segments
      auto issue_qk = [&](uint32_t g) -> bool {
        const uint32_t n = 2 * g, buf = n % R;
        const uint64_t k_desc = k_desc0 + buf * (TT::kTBytes >> 4);
        if (!tree_wait(&t_full[buf], (n / R) & 1)) { atomicCAS(p.err, 0u, 43u); return false; }
        tc::tc_fence_after();
#pragma unroll
        for (uint32_t hh = 0; hh < TT::kHalves; ++hh)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc::umma_f16(tmem_S + (g & 1) * RTN, q_desc + (hh * (128 * 128) + kk * 32) / 16, k_desc + (hh * (RTN * 128) + kk * 32) / 16, idesc_qk,
                         (hh | kk) ? 1u : 0u);
        tc::umma_commit(&t_empty[buf]);
        tc::umma_commit(&s_full[g & 1]);
        return true;
      };
      uint32_t g = 0, n_seg = 0;
      bool ok = true;
      for (; ok && seg.next(p); ++n_seg) {
        if (!tree_wait(q_full, n_seg & 1)) { atomicCAS(p.err, 0u, 42u); break; }
        ok = issue_qk(g);
        if (ok && seg.count == 1) tc::umma_commit(q_empty);
        for (uint32_t j = 0; j < seg.count && ok; ++j, ++g) {
          const uint32_t n = 2 * g + 1, buf = n % R;
          const uint64_t v_desc = v_desc0 + buf * (TT::kTBytes >> 4);
          // The next tile's scores are computed during this tile's softmax.  Their buffer holds P of the tile before, whose
          // product was issued before (the pipe runs in order), and the softmax left it when its p_ready arrived.
          if (j + 1 < seg.count) {
            if (!issue_qk(g + 1)) { ok = false; break; }
            if (j + 2 == seg.count) tc::umma_commit(q_empty);
          }
          if (!tree_wait(p_ready, g & 1)) { atomicCAS(p.err, 0u, 44u); ok = false; break; }
          if (!tree_wait(&t_full[buf], (n / R) & 1)) { atomicCAS(p.err, 0u, 45u); ok = false; break; }
          // a new segment's O overwrites the one before, which has to have been read
          if (j == 0 && n_seg > 0 && !tree_wait(o_free, (n_seg - 1) & 1)) { atomicCAS(p.err, 0u, 61u); ok = false; break; }
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc::umma_f16_ts(tmem_O, tmem_S + (g & 1) * RTN + kk * 8, v_desc + kk * 128, idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
          tc::umma_commit(&t_empty[buf]);
          tc::umma_commit(o_done);
        }
      }
    }
  } else {
    // ------------------------------ softmax + epilogue ------------------------------------
    const uint32_t quarter = warp & 3;
    const uint32_t r128 = quarter * 32 + lane;            // lane of the tile
    const uint32_t copy = (quarter * 32) / SPAN, r = r128 % SPAN;
    const uint32_t gh = r / p.lt, li = l0 + r - gh * p.lt;
    const bool row_valid = r < p.rows && li < a.l;
    const uint32_t lane_addr = (quarter * 32) << 16;
    const uint32_t tid = threadIdx.x - 64;
    bool ok = true;
    uint32_t g = 0, n_seg = 0;
    for (; seg.next(p); ++n_seg) {
      const uint32_t S = seg.skeys, cache_tiles = seg.of - (a.l + RTN - 1) / RTN;
      const unsigned char* mrow = a.mask + int64_t(seg.sb) * a.mask_sn + int64_t(row_valid ? li : 0) * a.mask_sl;
      int* odd = odd_flag + (n_seg & 1);
      float m_used = -INFINITY, l_run = 0.f;
      for (uint32_t j = 0; j < seg.count && ok; ++j, ++g) {
        const uint32_t t = seg.first + j;
        const bool drafted = t >= cache_tiles;
        const uint32_t key0 = (drafted ? t - cache_tiles : t) * RTN;
        const uint32_t nv = min(uint32_t(RTN), (drafted ? a.l : S) - key0);     // keys of the tile
        uint64_t vis = ~0ull;                                                   // this copy's columns the row sees
        if (drafted) {
          // read without a branch, so that the loads are under way together: past the last key, it again
          vis = 0;
          const unsigned char* mk = mrow + int64_t(key0) * a.mask_sk;
#pragma unroll 32
          for (int c = 0; c < NC; ++c) {
            const uint32_t k = copy * NC + c;
            const unsigned char seen = mk[int64_t(min(k, nv - 1)) * a.mask_sk];
            vis |= uint64_t(row_valid && k < nv && seen != 0) << c;
          }
        } else if (nv < RTN) {
          const int left = int(nv) - int(copy * NC);
          vis = left <= 0 ? 0ull : (left >= 64 ? ~0ull : (1ull << left) - 1ull);
        }
        if (!tree_wait_warp(&s_full[g & 1], (g >> 1) & 1)) { atomicCAS(p.err, 0u, 46u); ok = false; break; }
        tc::tc_fence_after();
        float sv[NC];
        const uint32_t s_addr = tmem_S + (g & 1) * RTN + lane_addr + copy * NC;
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
          const uint32_t n = 2 * g + 1, buf = n % R;
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
              bool bad = false;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                if ((e[x] & eb) == eb) { e[x] &= 0xFFFF0000u; bad = true; }
                if (((e[x] >> 16) & eb) == eb) { e[x] &= 0x0000FFFFu; bad = true; }
              }
              if (bad) { *at = w; *odd = 1; }
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
          if (!tree_wait_warp(o_done, (g - 1) & 1)) { atomicCAS(p.err, 0u, 48u); ok = false; break; }
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
        // The weights are rounded to the element type here (by half a step at most: 2^-8 of a weight in bf16, 2^-11 in fp16): the product takes both operands
        // in one type, and kuiops_sdpa does the same.  Their sum is taken before.  Against the definition in 64 bits a bf16 result
        // is off by 0.0018 to 0.0021 of its norm where rounding the result alone costs 0.0016 to 0.0017.  A second product with what the
        // rounding left off brings that back, but takes 4 % longer for 16 x 27 rows over 4000 keys and 21 % for 2 x 64 over 65000.
        // P over the scores it came from: column c holds keys 2 c and 2 c + 1, zero outside this copy's columns
        const uint32_t p_addr = tmem_S + (g & 1) * RTN + lane_addr;
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
      if (ok && !tree_wait_warp(o_done, (g - 1) & 1)) { atomicCAS(p.err, 0u, 49u); ok = false; }
      tc::tc_fence_after();

      // ---- the segment's rows: out when it is the whole unit, else a record ---------------------
      const bool whole = seg.count == seg.of;
      float mm = m_used, den = l_run, f = 1.f;
      if constexpr (REP > 1) {
        ml[r128] = make_float2(m_used, l_run);
        tree_barrier();
#pragma unroll
        for (int c = 0; c < REP; ++c) mm = fmaxf(mm, ml[c * SPAN + r].x);
        den = 0.f;
        // a copy whose scores were all NaN has no maximum but a NaN sum: the product keeps it
#pragma unroll
        for (int c = 0; c < REP; ++c) {
          const float2 x = ml[c * SPAN + r];
          den += x.y * (x.x == -INFINITY ? 1.f : fast_ex2(x.x - mm));
        }
        f = m_used == -INFINITY ? 1.f : fast_ex2(m_used - mm);
      } else {
        tree_barrier();                                    // the flag below is set by other warps
      }
      const bool bad = *odd != 0;
      const float inv = !whole ? 1.f : (den == 0.f ? 0.f : 1.f / den);
      const uint32_t rl = tree_record_floats(a.ev);
      float* recs = tree_tc_record(p.partials, a.ev, p.rows, p.row_tiles, range, seg.first == 0, rt, 0);
      // what was kept out of the product, for a row that sees it: columns c .. c + N - 1 of drafted position `pos`
      auto add_odd = [&](float* o, int N, uint32_t c, uint32_t pos) {
        const unsigned char* mr = a.mask + int64_t(seg.sb) * a.mask_sn + int64_t(pos) * a.mask_sl;
        const uint32_t t_hi = seg.first + seg.count, d_lo = seg.first > cache_tiles ? (seg.first - cache_tiles) * RTN : 0;
        const uint32_t d_hi = t_hi > cache_tiles ? min((t_hi - cache_tiles) * RTN, a.l) : 0;
        for (uint32_t k = d_lo; k < d_hi; ++k) {
          if (mr[int64_t(k) * a.mask_sk] == 0) continue;
          const T* v = static_cast<const T*>(a.DV) + int64_t(seg.sb) * a.dv_sn + int64_t(seg.skvh) * a.dv_sh + int64_t(k) * a.dv_sl + c;
#pragma unroll
          for (int x = 0; x < N; ++x) {
            const float y = c + x < a.ev ? ElemTraits<T>::to_f(v[x]) : 0.f;
            if (!isfinite(y)) o[x] += y;
          }
        }
      };
      auto out_row = [&](uint32_t hd, uint32_t pos) {
        return static_cast<T*>(a.out) + int64_t(seg.sb) * a.o_sn + int64_t(seg.skvh * p.G + hd) * a.o_sh + int64_t(pos) * a.o_sl;
      };
      if (ok && copy == 0 && row_valid) {
        if (!whole) *reinterpret_cast<float2*>(recs + size_t(r) * rl + rl - 4) = make_float2(mm, den);
        else if (a.lse)
          a.lse[(uint64_t(seg.sb) * a.h + seg.skvh * p.G + gh) * a.l + li] = den == 0.f ? -INFINITY : (mm + log2f(den)) * 0.6931471805599453f;
      }
      float odd_o = 0.f;                                   // NaN once an element of O was not finite
      if constexpr (REP == 1) {
        // a thread holds its row: 64 bytes of it at a time
        T* orow = out_row(gh, li);
        float* rrow = recs + size_t(r) * rl;
#pragma unroll 1
        for (uint32_t c0 = 0; c0 < DD; c0 += 32) {
          float ov[32];
          tc::tmem_ld32(tmem_O + lane_addr + c0, ov);
          tc::tmem_ld_wait();
          if (!ok || !row_valid) continue;
          odd_o += odd_test<32>(ov);
          if (bad) add_odd(ov, 32, c0, li);
          if (whole) {
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
              if (c0 + c >= a.ev) continue;
              *reinterpret_cast<uint4*>(orow + c0 + c) =
                  make_uint4(pack2<T>(ov[c] * inv, ov[c + 1] * inv), pack2<T>(ov[c + 2] * inv, ov[c + 3] * inv),
                             pack2<T>(ov[c + 4] * inv, ov[c + 5] * inv), pack2<T>(ov[c + 6] * inv, ov[c + 7] * inv));
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; c += 4)
              if (c0 + c < a.ev) *reinterpret_cast<float4*>(rrow + c0 + c) = make_float4(ov[c], ov[c + 1], ov[c + 2], ov[c + 3]);
          }
        }
        __syncwarp();
        tc::tc_fence_before();
        if (lane == 0) tc::mbar_arrive(o_free);
      } else {
        // The copies meet in shared memory, 16 columns at a time; a thread then owns four columns of one row (two rows, where
        // there are up to 64) throughout.
        constexpr int ITEMS = REP == 4 ? 1 : 2;
        T* orow[ITEMS];
        uint32_t irow[ITEMS], ipos[ITEMS];
        const uint32_t ic = (tid & 3) * 4;
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
          irow[x] = (tid >> 2) + x * 32;
          const uint32_t hd = irow[x] / p.lt;
          ipos[x] = l0 + irow[x] - hd * p.lt;
          if (irow[x] >= p.rows || ipos[x] >= a.l || !ok) irow[x] = 0xffffffffu;
          orow[x] = out_row(hd, ipos[x]);
        }
#pragma unroll 1
        for (uint32_t c0 = 0; c0 < DD; c0 += 16) {
          float ov[16];
          tc::tmem_ld16(tmem_O + lane_addr + c0, ov);
          tc::tmem_ld_wait();
          odd_o += odd_test<16>(ov);
          tree_barrier();                                  // the columns before have been taken, at first: every sum read
          if (c0 == 0) ml[r128].y = inv;                   // the row's factor, for the threads that write its columns
#pragma unroll
          for (int c = 0; c < 16; c += 4)
            *reinterpret_cast<float4*>(stage + r128 * 20 + c) = make_float4(ov[c] * f, ov[c + 1] * f, ov[c + 2] * f, ov[c + 3] * f);
          tree_barrier();
#pragma unroll
          for (int x = 0; x < ITEMS; ++x) {
            const uint32_t row = irow[x], c = c0 + ic;
            if (row == 0xffffffffu || c >= a.ev) continue;
            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < REP; ++k) {
              const float4 y = *reinterpret_cast<const float4*>(stage + (k * SPAN + row) * 20 + ic);
              o[0] += y.x; o[1] += y.y; o[2] += y.z; o[3] += y.w;
            }
            if (bad) add_odd(o, 4, c, ipos[x]);
            const float sc = ml[row].y;
            if (whole) *reinterpret_cast<uint2*>(orow[x] + c) = make_uint2(pack2<T>(o[0] * sc, o[1] * sc), pack2<T>(o[2] * sc, o[3] * sc));
            else *reinterpret_cast<float4*>(recs + size_t(row) * rl + c) = make_float4(o[0], o[1], o[2], o[3]);
          }
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(o_free);
      }
      if (tree_barrier_any(odd_o != 0.f) && ok) {
        OddSegment<T> sg;
        const uint32_t t_hi = seg.first + seg.count, k_lo = seg.first * RTN, k_hi = min(min(t_hi, cache_tiles) * RTN, S);
        sg.keys = k_hi > k_lo ? k_hi - k_lo : 0;
        sg.v = static_cast<const T*>(a.V) + int64_t(seg.sb) * a.v_sn + int64_t(seg.skvh) * a.v_sh + int64_t(k_lo) * a.v_ss;
        sg.dv = static_cast<const T*>(a.DV) + int64_t(seg.sb) * a.dv_sn + int64_t(seg.skvh) * a.dv_sh;
        sg.d_lo = seg.first > cache_tiles ? (seg.first - cache_tiles) * RTN : 0;
        sg.d_hi = t_hi > cache_tiles ? min((t_hi - cache_tiles) * RTN, a.l) : 0;
        sg.v_row = a.v_ss; sg.dv_row = a.dv_sl; sg.ev = a.ev;
        sg.mask = a.mask + int64_t(seg.sb) * a.mask_sn + int64_t(li) * a.mask_sl; sg.mask_sk = a.mask_sk;
        sg.row_on = copy == 0 && row_valid && den == den;          // a NaN among the row's scores is the row's own
        sg.out = out_row(gh, li);
        sg.rec = whole ? nullptr : recs + size_t(r) * rl;
        odd_patch<T>(sg);
      }
      if (tid == 0) *odd = 0;                              // this slot's next use is two segments away
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

struct TreeMerge { FastDiv by_chunks, by_heads, by_rows, by_lt; };

// Joins the records of the units that lie in several ranges.  WPR warps take two rows of one unit, side by side, warp w the records
// w, w + WPR, ..; lane c looks after the maximum and sum of its c-th record, every lane after four columns of all of them, the first four
// of which are on their way before the maxima are known.  The warps' results are added in warp order, so nothing depends on timing.
// (Four rows one after the other took 16 us where this takes a few: it is all latency.)
template <typename T, int WPR>
__global__ void __launch_bounds__(256)
sdpa_tree_tc_merge_kernel(const TreeTcParams p, const TreeMerge m) {
  constexpr int N = 2, A = 4;                              // rows of a warp, records ahead
  constexpr uint32_t PAIRS = 8 / WPR;                      // pairs of rows of a CTA
  const TreeArgs& a = p.a;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WPR;
  const uint32_t u = m.by_chunks.div(blockIdx.x), chunk = blockIdx.x - u * m.by_chunks.d, b = m.by_heads.div(u), kvh = u - b * a.h_kv;
  // The key counts are complete before the attention kernel's CTAs let this one start (each waited for them first); only the
  // records have to be waited for.
  const TreePlaces pl = tree_places(a, b);
  const uint32_t per = max((pl.all * a.h_kv + p.ranges - 1) / p.ranges, p.min_places), tiles = tree_tiles(a, tree_keys(a, b));
  const uint32_t begin = pl.before * a.h_kv + kvh * (tiles + kTreeLead) + kTreeLead;
  const uint32_t c0 = begin / per, pieces = (begin + tiles - 1) / per - c0 + 1;
  pdl_wait();
  pdl_trigger();
  if (pieces == 1) return;                                 // whole: written already
  const uint32_t rl = tree_record_floats(a.ev), tail = rl - 4, col = lane * 4;       // ev <= 128
  const size_t begins = size_t(p.row_tiles) * p.rows * rl, step = 2 * begins;        // from kind 0 to kind 1, and to the next range
  const bool on = col < a.ev;
  const uint32_t row0 = (chunk * PAIRS + warp / WPR) * N, all_rows = p.rows * p.row_tiles;
  const uint32_t mine = part < pieces ? (pieces - part + WPR - 1) / WPR : 0;         // records of this warp
  const float *x[N], *y[N];                                // the unit's first record, and the next ones', which are of kind 0
  uint32_t gh[N], li[N];
  float mm[N], den[N], acc[N][4];
  float4 ahead[N][A];
  float2 md[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t row = min(row0 + i, all_rows - 1), rt = m.by_rows.div(row), r = row - rt * p.rows;     // a row too many is read, not written
    gh[i] = m.by_lt.div(r);
    li[i] = row0 + i < all_rows ? rt * p.lt + r - gh[i] * p.lt : a.l;
    x[i] = tree_tc_record(p.partials, a.ev, p.rows, p.row_tiles, c0, 1, rt, r);
    y[i] = x[i] + begins;
    mm[i] = -INFINITY;
    den[i] = acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  }
  auto record = [&](int i, uint32_t k) {                    // this warp's k-th
    const uint32_t c = part + k * WPR;
    return c == 0 ? x[i] : y[i] + (c - 1) * step;
  };
  auto md_of = [&](int i, uint32_t k) {
    return k < mine ? __ldcg(reinterpret_cast<const float2*>(record(i, k) + tail)) : make_float2(-INFINITY, 0.f);
  };
  auto cols_of = [&](int i, uint32_t k) {
    return on && k < mine ? __ldcg(reinterpret_cast<const float4*>(record(i, k) + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
#pragma unroll
  for (int i = 0; i < N; ++i) md[i] = md_of(i, lane);
#pragma unroll
  for (int k = 0; k < A; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) ahead[i][k] = cols_of(i, k);
  for (uint32_t k0 = 0; k0 < mine; k0 += 32) {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (k0 > 0) md[i] = md_of(i, k0 + lane);
      const float mn = fmaxf(mm[i], warp_max(md[i].x));
      // without a maximum a record is zero, or NaN: the product keeps it
      f[i] = md[i].x == -INFINITY ? 1.f : fast_ex2(md[i].x - mn);
      const float g = mm[i] == -INFINITY ? 1.f : fast_ex2(mm[i] - mn);
      mm[i] = mn;
      den[i] = den[i] * g + warp_sum(f[i] * md[i].y);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] *= g;
    }
    for (uint32_t k = 0; k < min(32u, mine - k0); k += A) {
#pragma unroll
      for (int q = 0; q < A; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float fk = __shfl_sync(0xffffffffu, f[i], k + q);      // past the last record the columns are zero
          const float4 v = ahead[i][q];
          acc[i][0] = fmaf(fk, v.x, acc[i][0]); acc[i][1] = fmaf(fk, v.y, acc[i][1]);
          acc[i][2] = fmaf(fk, v.z, acc[i][2]); acc[i][3] = fmaf(fk, v.w, acc[i][3]);
          ahead[i][q] = cols_of(i, k0 + k + q + A);
        }
    }
  }
  if constexpr (WPR > 1) {
    __shared__ float join_s[8][N][32 * 4 + 2];
    float* mine_s = join_s[warp][0];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float* to = mine_s + i * (32 * 4 + 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e * 32 + lane] = acc[i][e];
      if (lane == 0) { to[128] = mm[i]; to[129] = den[i]; }
    }
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float top = -INFINITY;
      for (int w = 0; w < WPR; ++w) top = fmaxf(top, join_s[warp + w][i][128]);
      den[i] = acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      for (int w = 0; w < WPR; ++w) {
        const float* from = join_s[warp + w][i];
        const float f = from[128] == -INFINITY ? 1.f : fast_ex2(from[128] - top);
        den[i] = fmaf(f, from[129], den[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(f, from[e * 32 + lane], acc[i][e]);
      }
      mm[i] = top;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (li[i] >= a.l) continue;
    const uint32_t head = kvh * p.G + gh[i];
    if (on) {
      const float inv = den[i] == 0.f ? 0.f : 1.f / den[i];
      T* orow = static_cast<T*>(a.out) + int64_t(b) * a.o_sn + int64_t(head) * a.o_sh + int64_t(li[i]) * a.o_sl;
      *reinterpret_cast<uint2*>(orow + col) = make_uint2(pack2<T>(acc[i][0] * inv, acc[i][1] * inv), pack2<T>(acc[i][2] * inv, acc[i][3] * inv));
    }
    if (a.lse && lane == 0) a.lse[(uint64_t(b) * a.h + head) * a.l + li[i]] = den[i] == 0.f ? -INFINITY : (mm[i] + log2f(den[i])) * 0.6931471805599453f;
  }
}

bool sdpa_tree_tc_eligible(const TreeArgs& a) {
  if (a.dtype != KUIOPS_BF16 && a.dtype != KUIOPS_F16) return false;
  if (!(a.scale > 0.f)) return false;                       // the row maximum is taken before scaling
  if (a.e > 128 || a.ev > 128 || a.e % 8 || a.ev % 8) return false;
  if (a.h / a.h_kv > 128) return false;
  if (uint64_t(a.n) * a.h_kv * (uint64_t(a.s) / RTN + a.l / RTN + 2 + kTreeLead) >= (1ull << 31)) return false;
  // what a TMA descriptor takes: 16-byte aligned bases and strides
  auto ok = [&](const void* t, int64_t sn, int64_t sh, int64_t sl, uint32_t heads, uint32_t rows) {
    auto st = [](int64_t s) { return s > 0 && s % 8 == 0 && uint64_t(s) * 2 < (1ull << 40); };
    return aligned16(t) && (rows == 1 || st(sl)) && (heads == 1 || st(sh)) && (a.n == 1 || st(sn));
  };
  if (!ok(a.Q, a.q_sn, a.q_sh, a.q_sl, a.h, a.l) || !ok(a.out, a.o_sn, a.o_sh, a.o_sl, a.h, a.l)) return false;
  if (!ok(a.DK, a.dk_sn, a.dk_sh, a.dk_sl, a.h_kv, a.l) || !ok(a.DV, a.dv_sn, a.dv_sh, a.dv_sl, a.h_kv, a.l)) return false;
  return a.s == 0 || (ok(a.K, a.k_sn, a.k_sh, a.k_ss, a.h_kv, a.s) && ok(a.V, a.v_sn, a.v_sh, a.v_ss, a.h_kv, a.s));
}

struct TreeTcPlan { uint32_t lt, rows, row_tiles, ranges, min_places; };

static TreeTcPlan tree_tc_plan(const TreeArgs& a) {
  TreeTcPlan pl;
  const uint32_t G = a.h / a.h_kv, most = 128 / G;
  pl.row_tiles = (a.l + most - 1) / most;
  pl.lt = (a.l + pl.row_tiles - 1) / pl.row_tiles;
  pl.row_tiles = (a.l + pl.lt - 1) / pl.lt;
  pl.rows = G * pl.lt;
  // one range per resident CTA (two to an SM), none shorter than two tiles: below that joining costs more than it spreads
  pl.min_places = 2;
  const uint64_t slots = 2ull * num_sms() / pl.row_tiles;
  const uint64_t places = uint64_t(a.n) * a.h_kv * ((a.s + RTN - 1) / RTN + (a.l + RTN - 1) / RTN + kTreeLead);
  const uint64_t most_ranges = (places + pl.min_places - 1) / pl.min_places, ranges = slots < most_ranges ? slots : most_ranges;
  pl.ranges = ranges < 1 ? 1u : uint32_t(ranges);
  return pl;
}

size_t sdpa_tree_tc_workspace_bytes(const TreeArgs& a) {
  const TreeTcPlan pl = tree_tc_plan(a);
  return pl.ranges == 1 ? 0 : size_t(pl.ranges) * 2 * pl.row_tiles * pl.rows * tree_record_floats(a.ev) * sizeof(float);
}

template <typename T, int DD, int REP>
static int tree_tc_launch(const CUtensorMap* m, const TreeTcParams& p, cudaStream_t st) {
  auto kern = sdpa_tree_tc_kernel<T, DD, REP>;
  constexpr size_t smem = TreeTile<DD, REP>::kSmem;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KUIOPS_ELAUNCH;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return KUIOPS_ELAUNCH;
    configured.fetch_or(bit, std::memory_order_release);
  }
  const int rc = launch_pdl(kern, dim3(p.ranges * p.row_tiles), dim3(kTreeThreads), smem, st, m[0], m[1], m[2], m[3], m[4], p);
  if (rc != KUIOPS_OK || p.ranges == 1) return rc;
  // A unit has about ranges / units pieces.  More than eight are shared by eight warps (one unit of 64 rows, 65000 keys: 60 us with one
  // warp a pair of rows, 30 with eight); few are not worth meeting for.
  const uint32_t units = p.a.n * p.a.h_kv, wpr = p.ranges > 8 * units ? 8 : 1, pairs = 8 / wpr;
  const uint32_t chunks = (p.rows * p.row_tiles + 2 * pairs - 1) / (2 * pairs);      // n h l is below 2^31: checked with the shape
  TreeMerge mg;
  mg.by_chunks.set(chunks); mg.by_heads.set(p.a.h_kv); mg.by_rows.set(p.rows); mg.by_lt.set(p.lt);
  auto merge = wpr == 8 ? sdpa_tree_tc_merge_kernel<T, 8> : sdpa_tree_tc_merge_kernel<T, 1>;
  return launch_pdl(merge, dim3(units * chunks), dim3(256), 0, st, p, mg);
}

template <typename T, int DD>
static int tree_tc_launch_rep(const CUtensorMap* m, const TreeTcParams& p, cudaStream_t st) {
  if (p.rows <= 32) return tree_tc_launch<T, DD, 4>(m, p, st);
  if (p.rows <= 64) return tree_tc_launch<T, DD, 2>(m, p, st);
  return tree_tc_launch<T, DD, 1>(m, p, st);
}

int sdpa_tree_tc(const TreeArgs& a, cudaStream_t st) {
  const TreeTcPlan pl = tree_tc_plan(a);
  TreeTcParams p = {};
  p.a = a; p.G = a.h / a.h_kv; p.lt = pl.lt; p.rows = pl.rows; p.row_tiles = pl.row_tiles; p.ranges = pl.ranges; p.min_places = pl.min_places;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.partials = static_cast<float*>(a.workspace);
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
