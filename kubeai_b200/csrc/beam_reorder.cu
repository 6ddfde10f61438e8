// Tables, texts and partly filled pages of the beams that go on.
//
// A beam's whole pages never change again, so beams of one parent share them and only table rows move.  The page that is still being filled has one owner: a parent's
// first beam keeps it, and each further beam takes the page of a beam that nobody continues (there are as many), with the parent's rows copied into it.  Such a page is no one's
// source, so copies need no order among them, and no page is ever asked for.
// One launch: of a request's CTAs the first makes the tables and what becomes of its pages, the others find the parents for themselves and share texts and copies.
// Memory bounds it: 64 requests of 8 beams with 32 layers copy 339 MB in and out in 55.7 us, 6.1 TB/s.  One request of four beams is 5.8 us, six dependent trips (length, parents, table, page, rows,
// stores) behind a launch.
#include <cuda_runtime.h>

#include <algorithm>

#include "beam_step.h"
#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256, kColumns = 64, kBatch = 8;

__global__ void __launch_bounds__(kThreads)
beam_reorder_kernel(const b200_beam_reorder_args a) {
  __shared__ int parent[beam::kMaxBeams], page_of[beam::kMaxBeams], source[beam::kMaxBeams], target[beam::kMaxBeams];
  __shared__ int was[beam::kMaxBeams][kColumns];
  __shared__ int s_served, s_moves, s_common;
  __shared__ unsigned s_real;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, B = a.beams, row0 = s * B;
  griddep_enter();
  const int ctx = a.ctx[row0], full = ctx > 0 ? ctx / beam::kPage : 0, part = ctx > 0 ? ctx % beam::kPage : 0;
  if (tid < 32) {
    const int mine = lane < B ? a.parents[row0 + lane] : -1;
    const bool real = mine >= 0 && mine < B;
    const unsigned reals = __ballot_sync(0xffffffffu, real);
    const bool fits = ctx >= 0 && full + (part > 0) <= a.max_blocks;
    const bool served = __all_sync(0xffffffffu, lane >= B || a.ctx[row0 + lane] == ctx) && fits && reals;
    const int lead = __shfl_sync(0xffffffffu, mine, reals ? __ffs(reals) - 1 : 0);
    const int p = !served ? lane : real ? mine : lead;
    if (lane < B) parent[lane] = p;
    __syncwarp();
    beam::Heir h = {lane, lane};
    if (lane < B) h = beam::heir_of(parent, B, lane);
    if (lane < B) page_of[lane] = h.page;
    // the copies: from one page of the table's column to another
    bool moves = false;
    if (lane < B && served && part && h.page != h.parent) {
      const int from = a.block_tables[static_cast<size_t>(row0 + h.parent) * a.ld_tables + full], to = a.block_tables[static_cast<size_t>(row0 + h.page) * a.ld_tables + full];
      moves = from >= 0 && from < a.num_pages && to >= 0 && to < a.num_pages && from != to;
      if (moves) source[lane] = from, target[lane] = to;
    }
    const unsigned goes = __ballot_sync(0xffffffffu, moves);
    __syncwarp();
    const int from = moves ? source[lane] : 0, to = moves ? target[lane] : 0;
    __syncwarp();
    if (moves) {
      source[__popc(goes & ((1u << lane) - 1))] = from;
      target[__popc(goes & ((1u << lane) - 1))] = to;
    }
    if (lane == 0) {
      s_served = served;
      s_moves = __popc(goes);
      s_real = served ? reals : 0u;
      s_common = served ? full : 0;
    }
  }
  __syncthreads();
  const bool served = s_served;
  if (blockIdx.y == 0) {
    // ---- tables, and which whole pages nobody has any more
    for (int c0 = 0; c0 < a.max_blocks; c0 += kColumns) {
      const int cols = min(kColumns, a.max_blocks - c0);
      __syncthreads();
      for (int e = tid; e < B * kColumns; e += kThreads) {
        const int b = e / kColumns, c = e % kColumns;
        if (c < cols) was[b][c] = a.block_tables[static_cast<size_t>(row0 + b) * a.ld_tables + c0 + c];
      }
      __syncthreads();
      for (int e = tid; e < B * kColumns; e += kThreads) {
        const int i = e / kColumns, c = e % kColumns, column = c0 + c;
        if (c >= cols) continue;
        const int last = full + (part > 0);
        const int from = column < full ? parent[i] : column < last ? page_of[i] : i;
        a.tables_out[static_cast<size_t>(row0 + i) * a.ld_tables_out + column] = was[from][c];
        int gone = -1;
        if (served && column < full) {
          const int page = was[i][c];
          bool stays = false, named = false, alike = true;
          for (int b = 0; b < B; ++b) {
            stays = stays || was[parent[b]][c] == page;
            named = named || (b < i && was[b][c] == page);
            alike = alike && was[parent[b]][c] == was[parent[0]][c];
          }
          if (!stays && !named) gone = page;
          if (i == 0 && !alike) atomicMin(&s_common, column);
        }
        a.released[static_cast<size_t>(row0 + i) * a.max_blocks + column] = gone;
      }
    }
    __syncthreads();
    if (tid == 0) a.shared[s] = s_common * beam::kPage;
    return;
  }
  const int worker = blockIdx.y - 1, workers = gridDim.y - 1;
  // ---- texts
  if (a.texts) {
    for (int i = worker; i < B; i += workers) {
      const int p = parent[i], len = a.text_lens[row0 + p];
      const bool more = (s_real >> i & 1) && len >= 0 && len < a.room;
      const int* from = a.texts + static_cast<size_t>(row0 + p) * a.ld_texts;
      int* to = a.texts_out + static_cast<size_t>(row0 + i) * a.ld_texts_out;
      const int token = more ? a.tokens[row0 + i] : 0;
      for (int c = tid; c < a.room; c += kThreads) to[c] = more && c == len ? token : from[c];
      if (tid == 0) a.text_lens_out[row0 + i] = len + more;
    }
  }
  // ---- copies
  const int moves = s_moves, heads = 2 * a.kv_heads, rows = heads * part, piece = tid & 15;      // a head's rows lie one behind the other, 16 pieces of 16 bytes each
  const unsigned inverse = part > 1 ? 0xffffffffu / part + 1 : 0u;      // row / part = the upper half of row * inverse (parts below 16)
  for (int l = worker; l < a.layers && moves; l += workers) {
    uint4* kv = static_cast<uint4*>(a.kv) + static_cast<size_t>(l) * (a.layer_stride / 8);
    for (int m = 0; m < moves; ++m) {
      const uint4* from = kv + static_cast<size_t>(source[m]) * heads * 256 + piece;
      uint4* to = kv + static_cast<size_t>(target[m]) * heads * 256 + piece;
      for (int r0 = tid >> 4; r0 < rows; r0 += kBatch * (kThreads / 16)) {
        uint4 v[kBatch];
        auto at = [&](int k) {
          const int r = r0 + k * (kThreads / 16), head = part > 1 ? __umulhi(r, inverse) : r;
          return static_cast<size_t>(head) * 256 + (r - head * part) * 16;
        };
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (r0 + k * (kThreads / 16) < rows) v[k] = from[at(k)];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (r0 + k * (kThreads / 16) < rows) to[at(k)] = v[k];
      }
    }
  }
}

}  // namespace

int beam_reorder(const b200_beam_reorder_args& a, cudaStream_t st) {
  const int workers = std::min(std::max(a.layers, a.texts ? a.beams : 1), std::max(1, 16 * sm_count() / a.S));
  launch_pdl(beam_reorder_kernel, dim3(a.S, 1 + workers), dim3(kThreads), 0, st, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
