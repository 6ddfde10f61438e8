// Penalties, biases and grammar masks on logits, and the greedy choice, in one pass over the rows.
//
//   y = x;  said anywhere: y = y > 0 ? y / rho : y rho;  y -= phi c;  y -= pi where c > 0;  y += bias;  not allowed: -inf;  id = argmax y
//
// A vocabulary's rows are long and what is said about single tokens is short, so a cluster of CTAs shares a row: each keeps a table of its slice
// of the vocabulary in shared memory (how often a token was said, which bias entry it has), built once from the request's lists for all of the
// request's rows that the cluster takes, and a bit for every token that has an entry at all.  The pass over the logits then costs one load and three
// comparisons of pairs for eight tokens, and only tokens with their bit set are looked up.  Entries are initialised where a bit is set, so the
// table is never cleared as a whole.  A row's drafts are counted in ahead of it and out behind it.
// The slices' best pairs (value, token) meet through distributed shared memory.  Ties go to the lowest token: every comparison prefers it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "tree_step.h"
#include "umma2.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256, kMostCtas = 16, kRows = 256, kSlice = 8192, kMostSlice = 24576;
constexpr unsigned kPrompt = 0x80000000u;      // said in the prompt, which the repetition penalty alone counts

__device__ __forceinline__ unsigned long long peer_load(const void* p, unsigned rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_u32(smem_u32(p), rank)) : "memory");
  return v;
}

// (value, token) as one number that is larger for the better choice: the value's bits in ascending order, then the lower token.  Nothing: 0.
__device__ __forceinline__ unsigned long long packed(float y, int id) {
  if (id < 0) return 0;
  if (y == 0.f) y = 0.f;      // -0 is no smaller
  const unsigned u = __float_as_uint(y), up = u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(up) << 32 | static_cast<unsigned>(INT_MAX - id);
}

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const uint4& u, int j) {
    const unsigned w = j < 2 ? u.x : j < 4 ? u.y : j < 6 ? u.z : u.w;
    return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const uint4& u, int j) { return __uint_as_float(j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w); }
  static __device__ __forceinline__ float value(float v) { return v; }
};

__device__ __forceinline__ void store_one(__nv_bfloat16* p, float y) { *p = __float2bfloat16_rn(y); }
__device__ __forceinline__ void store_one(float* p, float y) { *p = y; }
struct None {};

// TIn: the logits; TOut: y kept, or None
template <typename TIn, typename TOut>
__global__ void __launch_bounds__(kThreads)
constrain_kernel(const b200_constrain_args a, int slice) {
  constexpr int N = Vec<TIn>::N;
  constexpr bool KEEP = !std::is_same<TOut, None>::value;
  extern __shared__ unsigned smem[];
  unsigned* count = smem;                                        // [slice]
  int* entry = reinterpret_cast<int*>(count + slice);            // [slice] the last bias entry, -1
  unsigned* known = reinterpret_cast<unsigned*>(entry + slice);  // [slice / 32 + 1] tokens with an entry
  __shared__ unsigned long long best_of[kRows];
  __shared__ unsigned long long warp_best[kThreads / 32];
  const int tid = threadIdx.x, rank = static_cast<int>(cluster_ctarank()), ctas = gridDim.x;
  const int lo = rank * slice, size = max(0, min(slice, a.V - lo));
  const int s = blockIdx.z, group = blockIdx.y, groups = gridDim.y;
  // ids may be read by a kernel behind this one ahead of its dependency wait: none is let in before the end
  griddep_wait();
  if (s == a.S) {      // rows that no request owns have no choice
    if (group || rank) return;
    bool plain = true;
    for (int i = tid; i < a.S; i += kThreads) plain = plain && a.starts[i] >= 0 && a.starts[i] <= a.starts[i + 1] && a.starts[i + 1] <= a.T;
    plain = __syncthreads_and(plain);
    for (int t = tid; t < a.T; t += kThreads) {
      bool owned = plain && t >= a.starts[0] && t < a.starts[a.S];
      for (int i = 0; !plain && !owned && i < a.S; ++i) owned = a.starts[i] >= 0 && a.starts[i + 1] <= a.T && t >= a.starts[i] && t < a.starts[i + 1];
      if (!owned) a.ids[t] = -1;
    }
    return;
  }
  int row0 = s, rows = 1;
  if (a.starts) {
    row0 = a.starts[s];
    const int end = a.starts[s + 1];
    rows = row0 >= 0 && end >= row0 && end <= a.T ? end - row0 : 0;
  }
  float rho = 1.f, pi = 0.f, phi = 0.f;
  if (a.penalties) rho = a.penalties[3 * s], pi = a.penalties[3 * s + 1], phi = a.penalties[3 * s + 2];
  int h0 = 0, h1 = 0, prompt = 0, b0 = 0, b1 = 0;
  if (a.history) {
    h0 = max(a.hist_starts[s], 0), h1 = min(a.hist_starts[s + 1], a.history_len);
    prompt = a.prompt_lens ? a.prompt_lens[s] : 0;
  }
  if (a.bias_starts) b0 = max(a.bias_starts[s], 0), b1 = min(a.bias_starts[s + 1], a.bias_len);
  if (group >= rows) rows = 0;      // (uniform over the cluster)

  // ---- the request's table
  for (int w = tid; w < slice / 32 + 1; w += kThreads) known[w] = 0;
  __syncthreads();
  auto know = [&](int v) {
    const int k = v - lo;
    if (k < 0 || k >= size) return;
    if (atomicOr(known + (k >> 5), 1u << (k & 31)) >> (k & 31) & 1) return;
    count[k] = 0;
    entry[k] = -1;
  };
  if (rows) {
    for (int i = h0 + tid; i < h1; i += kThreads) know(a.history[i]);
    for (int i = b0 + tid; i < b1; i += kThreads) know(a.bias_ids[i]);
    if (a.drafts)
      for (int i = tid; i < rows; i += kThreads) know(a.drafts[row0 + i]);
    __syncthreads();
    for (int i = h0 + tid; i < h1; i += kThreads) {
      const int k = a.history[i] - lo;
      if (k < 0 || k >= size) continue;
      if (i - h0 < prompt) atomicOr(count + k, kPrompt);
      else atomicAdd(count + k, 1u);
    }
    for (int i = b0 + tid; i < b1; i += kThreads) {
      const int k = a.bias_ids[i] - lo;
      if (k >= 0 && k < size) atomicMax(entry + k, i);
    }
    __syncthreads();
  }
  // the drafts that lead to row i, counted in or out
  auto drafted = [&](int i, unsigned by) {
    if (!a.masks) {
      for (int j = tid; j <= i; j += kThreads) {
        const int k = a.drafts[row0 + j] - lo;
        if (k >= 0 && k < size) atomicAdd(count + k, by);
      }
      return;
    }
    for (int j = tid; j < min(rows, 32 * a.words); j += kThreads) {
      if (!(static_cast<unsigned>(a.masks[static_cast<size_t>(row0 + i) * a.words + (j >> 5)]) >> (j & 31) & 1)) continue;
      const int k = a.drafts[row0 + j] - lo;
      if (k >= 0 && k < size) atomicAdd(count + k, by);
    }
  };

  // ---- the rows
  int done = 0;
  for (int i = group; i < rows; i += groups, ++done) {
    const int row = row0 + i;
    if (a.drafts) {
      drafted(i, 1u);
      __syncthreads();
    }
    const TIn* x = static_cast<const TIn*>(a.logits) + static_cast<size_t>(row) * a.ld;
    TOut* out = nullptr;
    if constexpr (KEEP) out = static_cast<TOut*>(a.out) + static_cast<size_t>(row) * a.ld_out;
    const unsigned* allow = nullptr;
    if (a.allow) {
      const int m = a.allow_rows ? a.allow_rows[row] : row;
      if (m >= 0 && m < a.allow_count) allow = reinterpret_cast<const unsigned*>(a.allow) + static_cast<size_t>(m) * a.ld_allow;
    }
    const int words = (a.V + 31) / 32;
    // whole vectors start where the row's addresses are multiples of 16 bytes: at tokens v with v + skew a multiple of N
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(x + lo) / sizeof(TIn) % N);
    float best = -INFINITY;
    int id = -1;
    for (int v0 = lo - skew + tid * N; v0 < lo + size; v0 += kThreads * N) {
      const int from = max(lo - v0, 0), to = min(lo + size - v0, N);      // this vector's tokens that are the slice's
      const unsigned inside = ((1u << to) - 1) & ~((1u << from) - 1);
      const int k0 = v0 + from - lo;                                      // of its first one, in the slice
      unsigned looked = __funnelshift_r(known[k0 >> 5], known[(k0 >> 5) + 1], k0 & 31) << from & inside;
      unsigned ok = inside;
      if (allow) {
        const int v = v0 + from, w = v >> 5;
        ok &= __funnelshift_r(allow[w], w + 1 < words ? allow[w + 1] : 0u, v & 31) << from;
      }
      if (!KEEP && !ok) continue;
      uint4 u;
      if (inside == (1u << N) - 1) {
        u = *reinterpret_cast<const uint4*>(x + v0);
      } else {
        TIn part[N] = {};
        for (int j = from; j < to; ++j) part[j] = x[v0 + j];
        u = *reinterpret_cast<const uint4*>(part);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (!(inside >> j & 1)) continue;
        float y = Vec<TIn>::get(u, j);
        if (looked >> j & 1) {
          const int k = v0 + j - lo;
          const unsigned c = count[k];
          if (c) y = y > 0.f ? __fdiv_rn(y, rho) : __fmul_rn(y, rho);
          const unsigned n = c & ~kPrompt;
          y = __fsub_rn(y, __fmul_rn(phi, static_cast<float>(n)));
          if (n) y = __fsub_rn(y, pi);
          if (entry[k] >= 0) y = __fadd_rn(y, a.bias_values[entry[k]]);
        }
        const bool allowed = ok >> j & 1;
        if constexpr (KEEP) store_one(out + v0 + j, allowed ? y : -INFINITY);
        if (allowed && (y > best || id < 0)) {
          best = y != y ? -INFINITY : y;
          id = v0 + j;
        }
      }
    }
    unsigned long long mine = packed(best, id);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((tid & 31) == 0) warp_best[tid >> 5] = mine;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kThreads / 32; ++w) mine = max(mine, warp_best[w]);
      best_of[done] = mine;
    }
    if (a.drafts) drafted(i, ~0u);
    __syncthreads();
  }

  // ---- the slices' best of each row
  if (!a.ids) return;
  __syncwarp();
  cluster_sync_all();
  for (int d = rank + ctas * tid; d < done; d += ctas * kThreads) {
    unsigned long long b = 0;
    for (int c = 0; c < ctas; ++c) b = max(b, peer_load(best_of + d, c));
    a.ids[row0 + group + d * groups] = b ? INT_MAX - static_cast<int>(static_cast<unsigned>(b)) : -1;
  }
  __syncwarp();
  cluster_sync_all();      // no CTA leaves while its best are read
}

template <typename TIn, typename TOut>
int launch(const b200_constrain_args& a, cudaStream_t st) {
  const auto kernel = constrain_kernel<TIn, TOut>;
  int ctas = 1;
  while (ctas < kMostCtas && (a.V + ctas - 1) / ctas > kSlice) ctas *= 2;
  const int slice = ((a.V + ctas - 1) / ctas + 31) / 32 * 32;
  const size_t smem = (2 * static_cast<size_t>(slice) + slice / 32 + 1) * 4;
  static std::atomic<unsigned long long> attr_done{0}, wide_done{0};
  if (!ensure_dynamic_smem(kernel, (2 * kMostSlice + kMostSlice / 32 + 1) * 4, &attr_done)) return -3;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -3;
  if (!(wide_done.load() >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return -3;
    wide_done.fetch_or(1ull << (dev & 63));
  }
  const int groups = a.starts ? std::max((a.T + kRows - 1) / kRows, std::min((a.T + a.S - 1) / a.S, 32)) : 1;
  if (groups > 65535) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, groups, a.S + (a.starts && a.ids ? 1 : 0));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, slice) == cudaSuccess ? 0 : -2;
}

}  // namespace

int constrain(const b200_constrain_args& a, cudaStream_t st) {
  if (a.logits_f32) return !a.out ? launch<float, None>(a, st) : a.out_f32 ? launch<float, float>(a, st) : launch<float, __nv_bfloat16>(a, st);
  return !a.out ? launch<__nv_bfloat16, None>(a, st) : a.out_f32 ? launch<__nv_bfloat16, float>(a, st) : launch<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace b200
