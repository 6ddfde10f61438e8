// Block tables, slots, positions and ancestor masks of a step, made on the device from the requests' lengths.
//
//   starts = running sum of rows;  need_s = pages(ctx + rows) - held;  off = running sum of need
//   a request is served while off + need <= pages left;  page(p) = p / 16 < held ? table[p / 16] : free[cursor + off + p / 16 - held]
//   slot(i) = page(ctx + i) * 16 + (ctx + i) % 16, -1 where the page's number is none;  ancestors(i) = {i} + ancestors(parent(i));  position(i) = ctx + |ancestors(i)| - 1
//
// What bounds it: the latency of a handful of dependent steps (lengths, two sums, a search, the stores), not bytes.  So one launch: every CTA
// of one cluster sums all requests' lengths for itself, which is cheaper than handing sums on, and then works on its share of rows
// and new pages, found by searching the sums (a request's rows may be one or thousands).  held and cursor may be written in place: the cluster
// barrier behind the sums is what lets them be.
// One request 4.5 us, 128 trees of up to 64 rows 6.8, 512 prompt portions of up to 127 rows (32642 rows) 11.2.
#include <cuda_runtime.h>
#include <limits.h>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "tree_step.h"
#include "umma2.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 1024, kCtas = 8;

__device__ __forceinline__ unsigned cluster_size() {
  unsigned n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
// Sum of v over the threads in front of this one (the block's whole sum in *all).  sums: 33 values of shared memory.
__device__ __forceinline__ long long block_sum_before(long long v, long long* sums, long long* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();      // the sums of the call before have been read
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < warps ? sums[lane] : 0;
    const long long own = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    sums[lane] = w - own;
    if (lane == 31) sums[32] = w;
  }
  __syncthreads();
  *all = sums[32];
  return sums[warp] + x - v;
}

__global__ void __launch_bounds__(kThreads)
step_maps_kernel(const b200_step_maps_args a) {
  extern __shared__ int smem[];
  int* s_start = smem;                    // [S + 1]
  int* s_off = s_start + a.S + 1;         // [S + 1] pages in front of each request's own
  int* s_held = s_off + a.S + 1;          // [S]
  unsigned char* s_flags = reinterpret_cast<unsigned char*>(s_held + a.S);
  __shared__ long long sums[33];
  __shared__ int s_short;                 // pages in front of the first request that finds too few
  const int tid = threadIdx.x;
  if (tid == 0) s_short = INT_MAX;
  // The kernels behind this one may read slots and positions ahead of their dependency wait, so none of them is let in before the end
  griddep_wait();
  const int first = min(max(a.cursor[0], 0), a.num_free);
  const int left = a.num_free - first;
  long long row_base = 0, page_base = 0;
  for (int base = 0; base < a.S; base += blockDim.x) {
    const int s = base + tid;
    int ctx = 0, n = 0, held = 0, need = 0, flags = 0;
    if (s < a.S) {
      ctx = a.ctx[s];
      n = a.rows[s];
      held = a.held[s];
    }
    long long all, before = row_base + block_sum_before(tree::rows_asked(n), sums, &all);
    row_base += all;
    if (s < a.S) {
      need = tree::pages_asked(ctx, n, held, a.max_blocks, a.words);
      if (need < 0 || before + n > a.T) {
        need = 0;
        flags = 2;
      }
      s_start[s] = static_cast<int>(min(before, static_cast<long long>(a.T)));
      s_held[s] = held;
    }
    before = page_base + block_sum_before(need, sums, &all);
    page_base += all;
    if (s < a.S) {
      if (need > 0 && before + need > left) {
        flags |= 1;
        atomicMin(&s_short, static_cast<int>(min(before, static_cast<long long>(INT_MAX))));
      }
      s_off[s] = static_cast<int>(min(before, static_cast<long long>(INT_MAX)));
      s_flags[s] = static_cast<unsigned char>(flags);
    }
  }
  if (tid == 0) {
    s_start[a.S] = static_cast<int>(min(row_base, static_cast<long long>(a.T)));
    s_off[a.S] = static_cast<int>(min(page_base, static_cast<long long>(INT_MAX)));
  }
  __syncthreads();
  const int taken = min(s_off[a.S], s_short);      // pages given out: every request in front of the first one that finds too few
  const int rank = static_cast<int>(cluster_ctarank()), stride = static_cast<int>(cluster_size() * blockDim.x), at = rank * blockDim.x + tid;
  for (int s = at; s <= a.S; s += stride) {
    a.starts[s] = s_start[s];
    if (s < a.S) a.status[s] = s_flags[s];
  }
  __syncwarp();
  cluster_sync_all();      // held and cursor have been read by all, status has been written
  for (int s = at; s < a.S; s += stride) {
    const int need = s_flags[s] ? 0 : s_off[s + 1] - s_off[s];
    a.held_out[s] = s_held[s] + need;
  }
  if (at == 0) a.cursor_out[0] = first + taken;
  for (int k = at; k < taken; k += stride) {
    const int s = tree::last_at_most(s_off, a.S, k);      // (requests that need none share the next one's offset)
    a.block_tables[static_cast<size_t>(s) * a.ld_tables + s_held[s] + (k - s_off[s])] = a.free_pages[first + k];
  }
  for (int t = at; t < a.T; t += stride) {
    int pos = 0, slot = -1, seq = -1;
    unsigned bits[tree::kMaxWords] = {};
    if (t < s_start[a.S]) {
      seq = tree::last_at_most(s_start, a.S, t);
      if (!s_flags[seq]) {
        const int i = t - s_start[seq], ctx = a.ctx[seq], p = ctx + i, page = p >> 4, held = s_held[seq];
        const int number = page < held ? a.block_tables[static_cast<size_t>(seq) * a.ld_tables + page] : a.free_pages[first + s_off[seq] + page - held];
        slot = tree::slot_on(number, p);
        int depth = i;
        bool odd = false;
        if (a.parents) {
          depth = -1;
          for (int j = i; j >= 0; ++depth) {
#pragma unroll
            for (int w = 0; w < tree::kMaxWords; ++w)
              if (w == j >> 5) bits[w] |= 1u << (j & 31);
            const int up = a.parents[s_start[seq] + j];
            odd |= up < -1 || up >= j;
            j = up >= 0 && up < j ? up : -1;
          }
        } else {
#pragma unroll
          for (int w = 0; w < tree::kMaxWords; ++w) bits[w] = i >= 32 * w + 31 ? 0xffffffffu : i >= 32 * w ? (2u << (i - 32 * w)) - 1 : 0;
        }
        if (odd) atomicOr(a.status + seq, 4);
        pos = ctx + depth;
      }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
    if (a.seqs) a.seqs[t] = seq;
#pragma unroll
    for (int w = 0; w < tree::kMaxWords; ++w)
      if (w < a.words) a.masks[static_cast<size_t>(t) * a.words + w] = static_cast<int>(bits[w]);
  }
}

}  // namespace

int step_maps(const b200_step_maps_args& a, cudaStream_t st) {
  const size_t smem = (3 * static_cast<size_t>(a.S) + 2) * sizeof(int) + a.S;
  static std::atomic<unsigned long long> attr_done{0};
  if (!ensure_dynamic_smem(step_maps_kernel, (3 * tree::kMaxRequests + 2) * sizeof(int) + tree::kMaxRequests, &attr_done)) return -3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCtas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {kCtas, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, step_maps_kernel, a) == cudaSuccess ? 0 : -2;
}

}  // namespace b200
