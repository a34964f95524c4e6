// The attention weight every key of a cache receives from a block of query rows, added up over the rows and over the
// heads that share the key:
//   out[b, kh, j] = mass[b, kh, j] + sum_{heads of kh} sum_{i: j < lim_i} exp(scale q_i . k_j - lse_i)
// with lse from the attention call that ran before.  Softmax weights need the final row sums, so they cannot leave the
// attention kernel in its one pass over the keys; this second pass reads K alone (no V) and needs no maximum.
//
// A key's sum is made by one thread in row order: no atomics, the result does not depend on timing.
#include "tree.cuh"

namespace kuiops {

static_assert(sizeof(kuiops_attn_mass_args) == 144, "callers pack the block without padding");

constexpr float kMassLog2e = 1.4426950408889634f;
constexpr int kMassRows = 16;                    // query rows a group stages at a time
constexpr int kMassAhead = 4;                    // rows of Q or K a warp has under way together

// Keys of entry b that row li counts for.
__device__ __forceinline__ uint32_t mass_limit(const MassArgs& p, uint32_t b, uint32_t li, uint32_t S) {
  if (p.q_lens) return clamp_len(p.q_lens[size_t(b % p.lens_n) * p.l + li], S);
  if (!p.is_causal) return S;
  return clamp_len((long long)li + 1 + (long long)S - (long long)p.l, S);
}

// SIMT form for every type, head dimension and stride: a thread owns a key, whose row the CTA keeps in shared memory (padded to
// an odd length: no bank conflicts), and dots it with sixteen query rows at a time, four features of them per broadcast load.
// `groups` parts of the CTA take the blocks of sixteen rows in turn and are added, in order, at the
// end.  fp32 arithmetic throughout; bound by shared-memory loads (20 for 64 multiply-adds; 192 rows over 3520 keys of eight
// KV heads of 128: 90 us, 15 TFLOP/s).
template <typename T>
__global__ void __launch_bounds__(256)
attn_mass_simt_kernel(const MassArgs p, uint32_t key_tiles, uint32_t groups) {
  extern __shared__ __align__(16) float sm[];
  const uint32_t KT = blockDim.x / groups, ep = ((p.e + 3) & ~3u) + 1, e4 = ep - 1;
  const uint32_t part = threadIdx.x / KT, t = threadIdx.x - part * KT, warp = t >> 5, warps = KT >> 5, lane = threadIdx.x & 31;
  float* q_s = sm + part * (kMassRows * (e4 + 2));              // [kMassRows][e4] of this part, then lse and limits
  float* lse_s = q_s + kMassRows * e4;
  uint32_t* lim_s = reinterpret_cast<uint32_t*>(lse_s + kMassRows);
  float* k_s = sm + groups * (kMassRows * (e4 + 2));    // [KT][ep]
  const uint32_t kt = blockIdx.x % key_tiles, u = blockIdx.x / key_tiles, kvh = u % p.h_kv, b = u / p.h_kv;
  const uint32_t G = p.h / p.h_kv, rows = G * p.l, key0 = kt * KT, j = key0 + t;
  pdl_wait();
  pdl_trigger();
  const uint32_t S = p.kv_lens ? clamp_len(p.kv_lens[b % p.lens_n], p.s) : p.s;
  float total = 0.f;
  if (key0 < S) {
    const T* Kb = static_cast<const T*>(p.K) + int64_t(b) * p.k_sn + int64_t(kvh) * p.k_sh;
    const uint32_t nk = min(KT, S - key0);
    const uint32_t all = blockDim.x >> 5;
    for (uint32_t r = threadIdx.x >> 5; r < nk; r += kMassAhead * all)      // loads of several rows under way together
      for (uint32_t c = lane; c < e4; c += 32) {
        float v[kMassAhead];
#pragma unroll
        for (int x = 0; x < kMassAhead; ++x)
          v[x] = r + x * all < nk && c < p.e ? ElemTraits<T>::to_f(Kb[int64_t(key0 + r + x * all) * p.k_ss + c]) : 0.f;
#pragma unroll
        for (int x = 0; x < kMassAhead; ++x)
          if (r + x * all < nk) k_s[(r + x * all) * ep + c] = v[x];
      }
    const float* krow = k_s + t * ep;
    const float qmul = p.scale * kMassLog2e;
    for (uint32_t r0 = part * kMassRows; r0 - part * kMassRows < rows; r0 += kMassRows * groups) {
      __syncthreads();
      // lanes 0 to 15 look up one row each; all lanes then copy the features of one row after the other
      const uint32_t row = r0 + (lane & (kMassRows - 1)), gh = row / p.l, li = row - gh * p.l;
      const int64_t off = int64_t(b) * p.q_sn + int64_t(kvh * G + gh) * p.q_sh + int64_t(li) * p.q_sl;
      if (warp == 0 && lane < kMassRows) {
        float ls = INFINITY;
        uint32_t lim = 0;
        if (row < rows) {
          ls = p.lse[(size_t(b) * p.h + kvh * G + gh) * p.l + li];
          // a row that saw nothing (-inf) or is not to be counted (+inf) has no weight to give
          if (!isinf(ls)) lim = mass_limit(p, b, li, S);
        }
        lse_s[lane] = ls * kMassLog2e;
        lim_s[lane] = lim;
      }
      for (uint32_t r = warp; r < kMassRows; r += kMassAhead * warps) {     // `warps` is 1 or 4: whole batches
        const T* q[kMassAhead];
#pragma unroll
        for (int x = 0; x < kMassAhead; ++x) q[x] = static_cast<const T*>(p.Q) + __shfl_sync(0xffffffffu, off, r + x * warps);
        for (uint32_t c = lane; c < e4; c += 32) {
          float v[kMassAhead];
#pragma unroll
          for (int x = 0; x < kMassAhead; ++x) v[x] = r0 + r + x * warps < rows && c < p.e ? ElemTraits<T>::to_f(q[x][c]) : 0.f;
#pragma unroll
          for (int x = 0; x < kMassAhead; ++x) q_s[(r + x * warps) * e4 + c] = v[x];
        }
      }
      __syncthreads();
      if (j < S) {
        float sc[kMassRows];
#pragma unroll
        for (int r = 0; r < kMassRows; ++r) sc[r] = 0.f;
        for (uint32_t c = 0; c < e4; c += 4) {
          const float k0 = krow[c], k1 = krow[c + 1], k2 = krow[c + 2], k3 = krow[c + 3];
#pragma unroll
          for (int r = 0; r < kMassRows; ++r) {
            const float4 q = *reinterpret_cast<const float4*>(q_s + r * e4 + c);
            sc[r] = fmaf(q.w, k3, fmaf(q.z, k2, fmaf(q.y, k1, fmaf(q.x, k0, sc[r]))));
          }
        }
        float w = 0.f;
#pragma unroll
        for (int r = 0; r < kMassRows; ++r)
          if (j < lim_s[r]) w += exp2f(fmaf(sc[r], qmul, -lse_s[r]));
        total += w;
      }
    }
  }
  __syncthreads();
  if (part > 0) sm[threadIdx.x] = total;                         // the staged rows are done with
  __syncthreads();
  if (part == 0 && j < p.s) {
    for (uint32_t g = 1; g < groups; ++g) total += sm[g * KT + t];
    const size_t o = (size_t(b) * p.h_kv + kvh) * p.s + j;
    p.out[o] = (p.mass ? p.mass[o] : 0.f) + total;
  }
}

constexpr size_t mass_simt_smem(uint32_t e, uint32_t keys, uint32_t groups) {
  const uint32_t e4 = (e + 3) & ~3u;
  return (size_t(groups) * kMassRows * (e4 + 2) + size_t(keys) * (e4 + 1)) * sizeof(float);
}
constexpr size_t mass_most(size_t a, size_t b) { return a > b ? a : b; }
// the widest head of each form below
constexpr size_t kMassSimtSmem = mass_most(mass_most(mass_simt_smem(256, 128, 2), mass_simt_smem(256, 32, 8)),
                                           mass_most(mass_simt_smem(512, 32, 4), mass_simt_smem(1024, 32, 1)));
static_assert(kMassSimtSmem <= 227 * 1024, "shared memory of an SM");

template <typename T>
static int mass_simt_launch(const MassArgs& a, cudaStream_t st) {
  // 128 keys and two parts; 32 keys and eight parts where that leaves SMs without work and there are rows to share (512 fp32 rows
  // of 64 features over 95 keys of six heads: 103 against 26 us).  Wider heads: 32 keys with as many parts as fit shared memory.
  const bool spread = a.h / a.h_kv * a.l > 32 && uint64_t(a.n) * a.h_kv * ((a.s + 127) / 128) < 4ull * num_sms();
  const uint32_t KT = a.e <= 256 && !spread ? 128 : 32, groups = a.e <= 256 ? (spread ? 8 : 2) : (a.e <= 512 ? 4 : 1);
  const uint32_t tiles = (a.s + KT - 1) / KT;
  const size_t smem = mass_simt_smem(a.e, KT, groups);
  auto kern = attn_mass_simt_kernel<T>;
  static std::atomic<uint64_t> configured{0};
  if (!raise_dynamic_smem(kern, kMassSimtSmem, configured)) return KUIOPS_ELAUNCH;
  const uint64_t grid = uint64_t(a.n) * a.h_kv * tiles;
  if (grid >= (1ull << 31)) return KUIOPS_ELIMIT;
  return launch_pdl(kern, dim3(unsigned(grid)), dim3(KT * groups), smem, st, a, tiles, groups);
}

int attn_mass_simt(const MassArgs& a, cudaStream_t st) {
  switch (a.dtype) {
    case KUIOPS_F32: return mass_simt_launch<float>(a, st);
    case KUIOPS_BF16: return mass_simt_launch<__nv_bfloat16>(a, st);
    default: return mass_simt_launch<__half>(a, st);
  }
}

}  // namespace kuiops

using namespace kuiops;

extern "C" {

int kuiops_attn_mass(const kuiops_attn_mass_args* args, kuiops_stream_t stream) {
  if (!args) return KUIOPS_EINVAL;
  MassArgs a = *args;
  if (a.dtype != KUIOPS_F32 && a.dtype != KUIOPS_BF16 && a.dtype != KUIOPS_F16) return KUIOPS_EINVAL;
  if (a.n == 0 || a.h == 0 || a.h_kv == 0 || a.l == 0 || a.s == 0 || a.e == 0 || a.h % a.h_kv) return KUIOPS_EINVAL;
  if (!a.Q || !a.K || !a.lse || !a.out || a.q_sl < int64_t(a.e) || a.k_ss < int64_t(a.e)) return KUIOPS_EINVAL;
  if ((a.kv_lens || a.q_lens) && (a.lens_n == 0 || a.n % a.lens_n)) return KUIOPS_EINVAL;
  if (!(a.scale - a.scale == 0.f)) return KUIOPS_EINVAL;
  if (a.e > 1024) return KUIOPS_EUNSUPPORTED;
  if (a.s > 0x7fffff00u || uint64_t(a.h / a.h_kv) * a.l >= (1ull << 31)) return KUIOPS_ELIMIT;
  if (a.lens_n == 0) a.lens_n = 1;
  return attn_mass_tc_eligible(a) ? attn_mass_tc(a, as_stream(stream)) : attn_mass_simt(a, as_stream(stream));
}

}  // extern "C"
