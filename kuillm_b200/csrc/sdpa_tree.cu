// Attention of l drafted tokens over a KV cache plus their own keys under an l x l mask:
//   out_i = sum_j w_ij v_j,   w_ij = exp(scale q_i . k_j - lse_i),   lse_i = log sum_j exp(scale q_i . k_j)
// over the cache keys j < kv_lens[b] and the drafted keys j with mask[b, i, j] != 0.  A masked key takes no part
// at all: whatever its row holds (infinities, NaN) reaches no output, and a row that sees nothing gives 0 / -inf.
//
// This file holds the entry point, the SIMT kernel for every type, head dimension and stride, and the kernel that
// joins key slices.  16-bit operands with up to 128 features per head run on the tensor cores (sdpa_tree_tc.cu).
#include "tree.cuh"
#include <mutex>

namespace kuiops {

static_assert(sizeof(kuiops_sdpa_tree_args) == 296, "callers pack the block without padding");

constexpr float kTreeLog2e = 1.4426950408889634f;
constexpr float kTreeLn2 = 0.6931471805599453f;
constexpr uint32_t kTreeMaxFeatures = 1024;      // of a query or key row

// SIMT form: a CTA owns R query rows of one (batch, KV head) and a slice of the 32-key tiles (cache tiles first, then
// the drafted ones).  Its four warps take tiles in turn; for the scores a lane owns a key and dots it with the R rows
// in shared memory, for the values a lane owns DV columns.  All arithmetic in fp32, softmax online in the log2 domain.
// Bound by shared-memory loads (64 x 64 fp32 rows over 4000 keys of eight KV heads: 665 us, 12.8 TFLOP/s); one row per KV head 25 us, latency.
template <typename T, int R, int DV>
__global__ void __launch_bounds__(128)
sdpa_tree_simt_kernel(const TreeArgs p, float* partials, uint32_t splits, uint32_t row_blocks, uint32_t e_pad) {
  extern __shared__ __align__(16) float sm[];
  constexpr int ACCW = DV * 32 + 2;
  float* q_s = sm;                                  // [R][e_pad]
  float* p_s = sm + R * e_pad + (threadIdx.x >> 5) * R * 32;      // this warp's weights, [R][32]
  float* mrg = sm + R * e_pad + 4 * R * 32;         // [4 warps][R][ACCW]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t split = blockIdx.x % splits;
  uint32_t u = blockIdx.x / splits;
  const uint32_t rb = u % row_blocks; u /= row_blocks;
  const uint32_t kvh = u % p.h_kv, b = u / p.h_kv;
  const uint32_t G = p.h / p.h_kv, rows = G * p.l;  // row = (head in group) * l + position
  pdl_wait();
  pdl_trigger();

  const float qmul = p.scale * kTreeLog2e;
  for (uint32_t i = tid; i < R * e_pad; i += 128) {
    const uint32_t row = rb * R + i / e_pad, c = i % e_pad;
    float v = 0.f;
    if (row < rows && c < p.e)
      v = ElemTraits<T>::to_f(static_cast<const T*>(p.Q)[int64_t(b) * p.q_sn + int64_t(kvh * G + row / p.l) * p.q_sh +
                                                         int64_t(row % p.l) * p.q_sl + c]);
    q_s[i] = v;
  }
  __syncthreads();

  const uint32_t S = p.kv_lens ? clamp_len(p.kv_lens[b], p.s) : p.s;
  const uint32_t cache_tiles = (S + 31) / 32, tiles = cache_tiles + (p.l + 31) / 32;
  const uint32_t per = (tiles + splits - 1) / splits;
  const uint32_t t_lo = min(split * per, tiles), t_hi = min(t_lo + per, tiles);
  const T* Kb = static_cast<const T*>(p.K) + int64_t(b) * p.k_sn + int64_t(kvh) * p.k_sh;
  const T* Vb = static_cast<const T*>(p.V) + int64_t(b) * p.v_sn + int64_t(kvh) * p.v_sh;
  const T* Kd = static_cast<const T*>(p.DK) + int64_t(b) * p.dk_sn + int64_t(kvh) * p.dk_sh;
  const T* Vd = static_cast<const T*>(p.DV) + int64_t(b) * p.dv_sn + int64_t(kvh) * p.dv_sh;
  const unsigned char* mk = p.mask + int64_t(b) * p.mask_sn;

  float m[R], lsum[R], acc[R][DV];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY; lsum[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DV; ++d) acc[r][d] = 0.f;
  }

  for (uint32_t t = t_lo + warp; t < t_hi; t += 4) {
    const bool drafted = t >= cache_tiles;
    const uint32_t key0 = drafted ? (t - cache_tiles) * 32 : t * 32;
    const uint32_t limit = drafted ? p.l : S;
    const uint32_t j = key0 + lane;
    const bool inside = j < limit;
    float sc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) sc[r] = 0.f;
    if (inside) {
      const T* krow = drafted ? Kd + int64_t(j) * p.dk_sl : Kb + int64_t(j) * p.k_ss;
      uint32_t c = 0;
      if ((reinterpret_cast<uintptr_t>(krow) & 15u) == 0) {
        constexpr int N = Vec16<T>::N, A = 4;          // four vectors of the row under way
        auto dot = [&](const Vec16<T>& kv, uint32_t at) {
          float kf[N];
#pragma unroll
          for (int x = 0; x < N; ++x) kf[x] = ElemTraits<T>::to_f(kv.v[x]);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float* q = q_s + r * e_pad + at;
#pragma unroll
            for (int x = 0; x < N; ++x) sc[r] = fmaf(q[x], kf[x], sc[r]);
          }
        };
        for (; c + A * N <= p.e; c += A * N) {
          Vec16<T> kv[A];
#pragma unroll
          for (int x = 0; x < A; ++x) kv[x] = ld16(krow + c + x * N);
#pragma unroll
          for (int x = 0; x < A; ++x) dot(kv[x], c + x * N);
        }
        for (; c + N <= p.e; c += N) dot(ld16(krow + c), c);
      }
      for (; c < p.e; ++c) {
        const float kf = ElemTraits<T>::to_f(krow[c]);
#pragma unroll
        for (int r = 0; r < R; ++r) sc[r] = fmaf(q_s[r * e_pad + c], kf, sc[r]);
      }
    }
    float pr[R];
    uint32_t vis[R];                                // keys of the tile that row r sees, one bit per key
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = rb * R + r;
      bool v = inside && row < rows;
      if (v && drafted) v = mk[int64_t(row % p.l) * p.mask_sl + int64_t(j) * p.mask_sk] != 0;
      vis[r] = __ballot_sync(0xffffffffu, v);
      const float s2 = v ? sc[r] * qmul : -INFINITY;
      const float mn = fmaxf(m[r], warp_max(s2));
      float corr = 1.f, pv = 0.f;
      if (mn != -INFINITY) corr = exp2f(m[r] - mn);            // m[r] = -inf gives 0
      if (v) pv = exp2f(s2 - (mn == -INFINITY ? 0.f : mn));     // a NaN score stays one
      lsum[r] = lsum[r] * corr + warp_sum(pv);
      m[r] = mn;
#pragma unroll
      for (int d = 0; d < DV; ++d) acc[r][d] *= corr;
      pr[r] = pv;
    }
    uint32_t any = 0, all = ~0u;
#pragma unroll
    for (int r = 0; r < R; ++r) { any |= vis[r]; all &= vis[r]; }
    __syncwarp();                                   // the weights of the tile before have been read
#pragma unroll
    for (int r = 0; r < R; ++r) p_s[r * 32 + lane] = pr[r];
    __syncwarp();
    // eight rows of V under way at a time (a loop over one row after the other is a chain of memory latencies: 76 against 25 us for
    // one row over 4000 keys)
    const uint32_t d0 = lane * DV;
    constexpr int B = DV == 8 ? 4 : 8;
    for (uint32_t j0 = 0; j0 < 32; j0 += B) {
      if (((any >> j0) & ((1u << B) - 1u)) == 0) continue;
      float vf[B][DV];
#pragma unroll
      for (int x = 0; x < B; ++x) {
        const uint32_t jj = j0 + x;
        const T* vrow = (drafted ? Vd + int64_t(key0 + jj) * p.dv_sl : Vb + int64_t(key0 + jj) * p.v_ss) + d0;
        const bool seen = (any >> jj) & 1u;              // rows that nobody sees are not read
        if (seen && d0 + DV <= p.ev && (reinterpret_cast<uintptr_t>(vrow) & (sizeof(T) * DV - 1)) == 0) {
          struct alignas(sizeof(T) * DV) Pack { T v[DV]; };
          const Pack w = *reinterpret_cast<const Pack*>(vrow);
#pragma unroll
          for (int d = 0; d < DV; ++d) vf[x][d] = ElemTraits<T>::to_f(w.v[d]);
        } else {
#pragma unroll
          for (int d = 0; d < DV; ++d) vf[x][d] = seen && d0 + d < p.ev ? ElemTraits<T>::to_f(vrow[d]) : 0.f;
        }
      }
      if (all == ~0u) {                             // every row sees every key of the tile
#pragma unroll
        for (int x = 0; x < B; x += 4) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float4 pj = *reinterpret_cast<const float4*>(p_s + r * 32 + j0 + x);
#pragma unroll
            for (int d = 0; d < DV; ++d)
              acc[r][d] = fmaf(pj.w, vf[x + 3][d], fmaf(pj.z, vf[x + 2][d], fmaf(pj.y, vf[x + 1][d], fmaf(pj.x, vf[x][d], acc[r][d]))));
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < B; ++x) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float pj = p_s[r * 32 + j0 + x];
            if ((vis[r] >> (j0 + x)) & 1u) {
#pragma unroll
              for (int d = 0; d < DV; ++d) acc[r][d] = fmaf(pj, vf[x][d], acc[r][d]);
            }
          }
        }
      }
    }
  }

  // join the four warps in warp order
  {
    float* mine = mrg + size_t(warp) * R * ACCW;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int d = 0; d < DV; ++d) mine[r * ACCW + lane * DV + d] = acc[r][d];
      if (lane == 0) { mine[r * ACCW + DV * 32] = m[r]; mine[r * ACCW + DV * 32 + 1] = lsum[r]; }
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < R * p.ev; i += 128) {
    const uint32_t r = i / p.ev, c = i % p.ev, row = rb * R + r;
    if (row >= rows) continue;
    float mm = -INFINITY;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, mrg[(w * R + r) * ACCW + DV * 32]);
    float a = 0.f, den = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float* rec = mrg + (w * R + r) * ACCW;
      const float f = rec[DV * 32] == -INFINITY ? 0.f : exp2f(rec[DV * 32] - mm);
      // a slice whose scores were all NaN has no maximum but a NaN sum: the product keeps it
      a += f * rec[c]; den += f * rec[DV * 32 + 1];
    }
    const uint32_t head = kvh * G + row / p.l, li = row % p.l;
    const uint64_t orow = (uint64_t(b) * p.h + head) * p.l + li;
    if (splits == 1) {
      static_cast<T*>(p.out)[int64_t(b) * p.o_sn + int64_t(head) * p.o_sh + int64_t(li) * p.o_sl + c] =
          ElemTraits<T>::from_f(den == 0.f ? 0.f : a / den);
      if (c == 0 && p.lse) p.lse[orow] = den == 0.f ? -INFINITY : (mm + log2f(den)) * kTreeLn2;
    } else {
      float* rec = tree_record(partials, orow, splits, split, p.ev);
      rec[c] = a;
      if (c == 0) { rec[tree_record_floats(p.ev) - 4] = mm; rec[tree_record_floats(p.ev) - 3] = den; }
    }
  }
}

// One warp per output row: the slices' records are added in slice order, so the result does not depend on timing.
template <typename T>
__global__ void __launch_bounds__(128)
sdpa_tree_merge_kernel(const TreeArgs p, const float* partials, uint32_t splits) {
  const uint64_t row = uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (row >= uint64_t(p.n) * p.h * p.l) return;
  const uint32_t rl = tree_record_floats(p.ev);
  const float* base = partials + row * splits * rl;
  float mm = -INFINITY;
  for (uint32_t s = lane; s < splits; s += 32) mm = fmaxf(mm, __ldcg(base + size_t(s) * rl + rl - 4));
  mm = warp_max(mm);
  const uint32_t li = uint32_t(row % p.l), head = uint32_t(row / p.l % p.h), b = uint32_t(row / (uint64_t(p.l) * p.h));
  T* orow = static_cast<T*>(p.out) + int64_t(b) * p.o_sn + int64_t(head) * p.o_sh + int64_t(li) * p.o_sl;
  float den = 0.f;
  for (uint32_t c0 = 0; c0 < p.ev; c0 += 128) {
    const uint32_t c = c0 + lane * 4;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    den = 0.f;
#pragma unroll 4
    for (uint32_t s = 0; s < splits; ++s) {
      const float* rec = base + size_t(s) * rl;
      const float mw = __ldcg(rec + rl - 4), lw = __ldcg(rec + rl - 3);
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - mm);
      den += f * lw;
      if (c < p.ev) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(rec + c));
        acc[0] += f * x.x; acc[1] += f * x.y; acc[2] += f * x.z; acc[3] += f * x.w;
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (c + x < p.ev) orow[c + x] = ElemTraits<T>::from_f(den == 0.f ? 0.f : acc[x] / den);
  }
  if (p.lse && lane == 0) p.lse[row] = den == 0.f ? -INFINITY : (mm + log2f(den)) * kTreeLn2;
}

template <typename T, int R, int DV>
static int simt_launch(const TreeArgs& a, float* partials, uint32_t splits, cudaStream_t st) {
  const uint32_t e_pad = (a.e + 3) & ~3u, rows = a.h / a.h_kv * a.l, row_blocks = (rows + R - 1) / R;
  constexpr size_t fixed = (size_t(4) * R * 32 + size_t(4) * R * (DV * 32 + 2)) * sizeof(float);
  const size_t smem = fixed + size_t(R) * e_pad * sizeof(float);
  auto kern = sdpa_tree_simt_kernel<T, R, DV>;
  static std::atomic<uint64_t> configured{0};
  if (!raise_dynamic_smem(kern, fixed + size_t(R) * kTreeMaxFeatures * sizeof(float), configured)) return KUIOPS_ELAUNCH;
  const uint64_t grid = uint64_t(a.n) * a.h_kv * row_blocks * splits;
  if (grid >= (1ull << 31)) return KUIOPS_ELIMIT;
  return launch_pdl(kern, dim3(unsigned(grid)), dim3(128), smem, st, a, partials, splits, row_blocks, e_pad);
}

template <typename T>
static int simt_launch_t(const TreeArgs& a, float* partials, uint32_t splits, cudaStream_t st) {
  const bool few = a.h / a.h_kv * a.l <= 4;
  if (a.ev <= 64) return few ? simt_launch<T, 4, 2>(a, partials, splits, st) : simt_launch<T, 8, 2>(a, partials, splits, st);
  if (a.ev <= 128) return few ? simt_launch<T, 4, 4>(a, partials, splits, st) : simt_launch<T, 8, 4>(a, partials, splits, st);
  return few ? simt_launch<T, 4, 8>(a, partials, splits, st) : simt_launch<T, 8, 8>(a, partials, splits, st);
}

// Slices per (batch, KV head, row block): as many CTAs as two waves hold (a 128-thread CTA, four to an SM), with at least
// four 32-key tiles each, one per warp.
uint32_t sdpa_tree_simt_splits(const TreeArgs& a) {
  const uint32_t rows = a.h / a.h_kv * a.l, R = rows <= 4 ? 4 : 8;
  const uint64_t units = uint64_t(a.n) * a.h_kv * ((rows + R - 1) / R), want = 8ull * num_sms() / units;
  const uint32_t cap = (a.s / 32 + (a.l + 31) / 32) / 4;
  const uint64_t v = want < cap ? want : cap;
  return v < 1 ? 1u : (v > 64 ? 64u : uint32_t(v));
}

int sdpa_tree_simt(const TreeArgs& a, float* partials, uint32_t splits, cudaStream_t st) {
  switch (a.dtype) {
    case KUIOPS_F32: return simt_launch_t<float>(a, partials, splits, st);
    case KUIOPS_BF16: return simt_launch_t<__nv_bfloat16>(a, partials, splits, st);
    default: return simt_launch_t<__half>(a, partials, splits, st);
  }
}

int sdpa_tree_merge(const TreeArgs& a, const float* partials, uint32_t splits, cudaStream_t st) {
  const uint64_t grid = (uint64_t(a.n) * a.h * a.l + 3) / 4;
  if (grid >= (1ull << 31)) return KUIOPS_ELIMIT;
  switch (a.dtype) {
    case KUIOPS_F32: return launch_pdl(sdpa_tree_merge_kernel<float>, dim3(unsigned(grid)), dim3(128), 0, st, a, partials, splits);
    case KUIOPS_BF16: return launch_pdl(sdpa_tree_merge_kernel<__nv_bfloat16>, dim3(unsigned(grid)), dim3(128), 0, st, a, partials, splits);
    default: return launch_pdl(sdpa_tree_merge_kernel<__half>, dim3(unsigned(grid)), dim3(128), 0, st, a, partials, splits);
  }
}

}  // namespace kuiops

using namespace kuiops;

static int tree_shape(int dtype, uint32_t n, uint32_t h, uint32_t h_kv, uint32_t l, uint32_t s, uint32_t e, uint32_t ev) {
  if (dtype != KUIOPS_F32 && dtype != KUIOPS_BF16 && dtype != KUIOPS_F16) return KUIOPS_EINVAL;
  if (n == 0 || h == 0 || h_kv == 0 || l == 0 || e == 0 || ev == 0 || h % h_kv) return KUIOPS_EINVAL;
  if (e > kTreeMaxFeatures || ev > 256) return KUIOPS_EUNSUPPORTED;
  if (l > KUIOPS_TREE_MAX_ROWS || s > 0x7fffff00u || uint64_t(n) * h * l >= (1ull << 31)) return KUIOPS_ELIMIT;
  return KUIOPS_OK;
}

static size_t tree_record_bytes(const TreeArgs& a, uint32_t splits) {
  return splits <= 1 ? 0 : size_t(a.n) * a.h * a.l * splits * tree_record_floats(a.ev) * sizeof(float);
}

static bool tree_tc_shape(const TreeArgs& a) { return a.dtype != KUIOPS_F32 && a.e <= 128 && a.ev <= 128 && a.h / a.h_kv <= 128; }

extern "C" {

size_t kuiops_sdpa_tree_workspace_bytes(int dtype, uint32_t n, uint32_t h, uint32_t h_kv, uint32_t l, uint32_t s, uint32_t e,
                                        uint32_t ev) {
  TreeArgs a = {};
  if (tree_shape(dtype, n, h, h_kv, l, s, e, ev) != KUIOPS_OK) return 0;
  a.dtype = dtype; a.n = n; a.h = h; a.h_kv = h_kv; a.l = l; a.s = s; a.e = e; a.ev = ev;
  // which kernel runs also depends on alignment, unknown here: cover both
  const size_t simt = tree_record_bytes(a, sdpa_tree_simt_splits(a)), tc = tree_tc_shape(a) ? sdpa_tree_tc_workspace_bytes(a) : 0;
  return simt > tc ? simt : tc;
}

int kuiops_sdpa_tree(const kuiops_sdpa_tree_args* args, kuiops_stream_t stream) {
  if (!args) return KUIOPS_EINVAL;
  const TreeArgs& a = *args;
  const int rc = tree_shape(a.dtype, a.n, a.h, a.h_kv, a.l, a.s, a.e, a.ev);
  if (rc != KUIOPS_OK) return rc;
  if (!a.Q || !a.DK || !a.DV || !a.mask || !a.out || (a.s > 0 && (!a.K || !a.V))) return KUIOPS_EINVAL;
  const int64_t e = a.e, ev = a.ev;
  if (a.q_sl < e || a.dk_sl < e || a.dv_sl < ev || a.o_sl < ev) return KUIOPS_EINVAL;
  if (a.s > 0 && (a.k_ss < e || a.v_ss < ev)) return KUIOPS_EINVAL;
  if (a.mask_sn < 0 || a.mask_sl < 0 || a.mask_sk < 0) return KUIOPS_EINVAL;
  if (!(a.scale - a.scale == 0.f)) return KUIOPS_EINVAL;          // a finite number
  cudaStream_t st = as_stream(stream);
  const bool tc = sdpa_tree_tc_eligible(a);
  const uint32_t splits = sdpa_tree_simt_splits(a);
  const size_t need = tc ? sdpa_tree_tc_workspace_bytes(a) : tree_record_bytes(a, splits);
  if (need && (!a.workspace || a.workspace_bytes < need || !aligned16(a.workspace))) return KUIOPS_EWORKSPACE;
  // A call's kernels follow each other in the stream: host threads that share a stream share its workspace, and another call's
  // kernel between these two would overwrite the records.
  static std::mutex launches;
  std::unique_lock<std::mutex> lock(launches, std::defer_lock);
  if (need) lock.lock();
  if (tc) return sdpa_tree_tc(a, st);
  float* partials = static_cast<float*>(a.workspace);
  const int run = sdpa_tree_simt(a, partials, splits, st);
  if (run != KUIOPS_OK || splits == 1) return run;
  return sdpa_tree_merge(a, partials, splits, st);
}

}  // extern "C"
