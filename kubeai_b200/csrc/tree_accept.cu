// The drafts that the choices confirm, and their cache rows moved to where they stay.
//
//   path_0 = 0;  path_{k+1} = the lowest row i whose parent is path_k and whose draft is ids[path_k];  K, V at ctx + path_k -> ctx + k, every layer
//
// A row knows by itself whether its parent's choice confirms it, so the rows look in parallel, the lowest confirmed child of each
// row is a minimum in shared memory, and the path is a chase through it.  Every CTA finds its request's path for itself (rows of a few hundred
// bytes in L2) and moves it in its own layers, so the operation is one launch.  A path ascends and never runs ahead of itself (path_k >= k): a thread that
// moves the same 16 bytes of all the path's rows in order overwrites nothing that it has still to read, and no other thread reads those.
// What bounds it: the chain lengths, parents, choices, path, tables, rows, five trips to memory one behind the other (one request 3.2 us); behind it the bytes moved
// (64 requests of up to 48 rows, 32 layers: 40 MB in and out in 9.6 us, 4.2 TB/s of the whole call).
#include <cuda_runtime.h>
#include <limits.h>

#include <algorithm>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "tree_step.h"

namespace b200 {
namespace {

constexpr int kThreads = 256, kMostPath = 256, kBatch = 8;

__global__ void __launch_bounds__(kThreads)
tree_accept_kernel(const b200_tree_accept_args a) {
  __shared__ int child[tree::kMaxTree];
  __shared__ int path[kMostPath];
  __shared__ long long move_to[kMostPath], move_from[kMostPath];      // cache rows
  __shared__ int s_len, s_moves;
  const int s = blockIdx.x, tid = threadIdx.x;
  // new lengths and tokens may be read by a kernel behind this one ahead of its dependency wait: none is let in before the end
  griddep_wait();
  const tree::Request r = tree::request_of(a.starts, a.ctx, s, a.T, a.max_blocks, tree::kMaxTree, a.status);
  for (int i = tid; i < r.rows; i += kThreads) child[i] = INT_MAX;
  __syncthreads();
  for (int i = tid; i < r.rows; i += kThreads) {
    const int p = tree::parent_of(a.parents, r.row0, i);
    if (p < 0) continue;
    const int chosen = a.ids[r.row0 + p];
    if (chosen >= 0 && chosen == a.drafts[r.row0 + i]) atomicMin(child + p, i);
  }
  __syncthreads();
  if (tid == 0) {
    int len = 0;
    for (int at = 0; r.rows > 0 && at != INT_MAX && len < a.max_path; at = child[at]) path[len++] = at;
    s_len = len;
  }
  __syncthreads();
  const int len = s_len;
  if (blockIdx.y == 0) {
    for (int k = tid; k < a.max_path; k += kThreads) {
      a.path[static_cast<size_t>(s) * a.max_path + k] = k < len ? path[k] : -1;
      a.tokens[static_cast<size_t>(s) * a.max_path + k] = k < len ? a.ids[r.row0 + path[k]] : -1;
    }
    if (tid == 0) {
      a.accepted[s] = len;
      a.new_ctx[s] = a.ctx[s] + len;
    }
  }
  // what moves, in order
  const int* table = a.block_tables + static_cast<size_t>(s) * a.ld_tables;
  if (tid < 32) {
    int moves = 0;
    for (int k0 = 0; k0 < len; k0 += 32) {
      const int k = k0 + tid;
      long long from = -1, to = -1;
      if (k < len && path[k] != k) {
        from = tree::cache_row(table, r.ctx + path[k], a.num_pages);
        to = tree::cache_row(table, r.ctx + k, a.num_pages);
      }
      const unsigned goes = __ballot_sync(0xffffffffu, from >= 0 && to >= 0);
      if (from >= 0 && to >= 0) {
        const int m = moves + __popc(goes & ((1u << tid) - 1));
        move_from[m] = from;
        move_to[m] = to;
      }
      moves += __popc(goes);
    }
    if (tid == 0) s_moves = moves;
  }
  __syncthreads();
  const int moves = s_moves;
  if (!moves) return;
  const int heads = a.kv_heads, tasks = 2 * heads * 16;      // 16-byte pieces of a token's K and V rows
  for (int l = blockIdx.y; l < a.layers; l += gridDim.y) {
    uint4* kv = static_cast<uint4*>(a.kv) + static_cast<size_t>(l) * (a.layer_stride / 8);
    for (int task = tid; task < tasks; task += kThreads) {
      const int piece = task & 15, row = task >> 4;          // row: K heads, then V heads
      auto place = [&](long long cache_row) { return ((cache_row >> 4) * 2 * heads + row) * 256 + (cache_row & 15) * 16 + piece; };
      for (int m = 0; m < moves; m += kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (m + j < moves) v[j] = kv[place(move_from[m + j])];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (m + j < moves) kv[place(move_to[m + j])] = v[j];
      }
    }
  }
}

}  // namespace

int tree_accept(const b200_tree_accept_args& a, cudaStream_t st) {
  // As many CTAs as the SMs hold, four each: more of them find their paths in vain (64 requests, 32 layers: 9.6 us, with two an SM 13.7, with sixteen 12.6)
  const int parts = std::min(std::max(a.layers, 1), std::max(1, 4 * sm_count() / a.S));
  launch_pdl(tree_accept_kernel, dim3(a.S, parts), dim3(kThreads), 0, st, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
