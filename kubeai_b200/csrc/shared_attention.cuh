// What the two halves of the kernel of shared_attention.cu have in common: which rows and keys an item has, and where its rows go.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "beam_step.h"
#include "ptx.cuh"

namespace b200 {
namespace shared_attn {

using beam::Lengths;
using beam::Part;
typedef __nv_bfloat16 bf16;
constexpr int kD = 128, kTile16 = 16, kNarrow = 2 * kTile16;
// kNarrow: rows (token * group + head) of a part that go to narrow CTAs, whose warps have tiles of 16.  64 groups of 32 rows behind up to 450 tokens take 62.9 us there and 82.7 in wide CTAs, 8 behind up to
// 4000 40.2 and 39.3; of 48 rows, in teams of four warps, 114 us behind 4000 and 43 in wide CTAs, 64 groups behind 450 137 and 101.
constexpr int kLd = kD + 4;                // floats from row to row of the workspace: output, maximum, sum
constexpr int kWaitLimit = 1 << 22;

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_limited(bar, parity, kWaitLimit)); }
// two bf16 without infinities and NaN
__device__ __forceinline__ uint32_t without_odd(uint32_t u) { return ((u & 0x7f80u) == 0x7f80u ? 0u : u & 0xffffu) | ((u & 0x7f800000u) == 0x7f800000u ? 0u : u & 0xffff0000u); }

// Where the rows of a token and key head are: their own keys' part, and what their group shares.
struct Place {
  int slot, parts;      // parts 0: in the rows of all (or in the output), else in the slots of `parts` ranges, slot the first: of kWideRows rows, or of 16 and a team's tiles
  int row;              // the token's first row there
  int flags;
};
constexpr int kJoined = 1, kTeam = 4;      // own rows: the group's are to be added; times the team, 0 for a wide CTA
struct Space {
  Place* places;        // [2][T][kv_heads]: the groups', the requests' own
  float* narrow;        // [warps][2][16][kLd], a team's warps together: a range's first item, which another range began, and its last
  float* wide;          // [CTAs][2][kWideRows][kLd], the same
  float* rows;          // [2][T][q_heads][kLd]
};
struct Sizes {
  int warps, ctas;      // of all CTAs, which may all be narrow, and how many may be wide
};
constexpr int kWideRows = 256;      // rows of an item of a wide CTA
__host__ __device__ inline Space space_of(const b200_shared_attn_args& a, const Sizes& n) {
  Space s;
  s.places = static_cast<Place*>(a.workspace);
  s.narrow = reinterpret_cast<float*>(s.places + 2ll * a.T * a.kv_heads);
  s.wide = s.narrow + static_cast<long long>(n.warps) * 2 * kTile16 * kLd;
  s.rows = s.wide + static_cast<long long>(n.ctas) * 2 * kWideRows * kLd;
  return s;
}

// The lengths, in shared memory where they fit: parts are looked up by chains of dependent loads, at the head of a kernel and at every item's beginning.  With a barrier behind it; `groups`
// where they are wanted.
constexpr int kStaged = 256;
struct Staged {
  int starts[kStaged + 1], ctx[kStaged], status[kStaged], group_starts[kStaged + 1], shared[kStaged];
};
__device__ __forceinline__ Lengths lengths_of(const b200_shared_attn_args& a, Staged* to, int tid, int threads) {
  Lengths n = {a.starts, a.ctx, a.group_starts, a.shared, a.status, a.S, a.T, a.G, a.max_blocks, a.max_rows};
  if (a.S <= kStaged && a.G <= kStaged) {
    for (int s = tid; s <= a.S; s += threads) {
      to->starts[s] = a.starts[s];
      if (s < a.S) to->ctx[s] = a.ctx[s];
      if (s < a.S && a.status) to->status[s] = a.status[s];
    }
    if (a.G)
      for (int g = tid; g <= a.G; g += threads) {
        to->group_starts[g] = a.group_starts[g];
        if (g < a.G) to->shared[g] = a.shared[g];
      }
    n.starts = to->starts; n.ctx = to->ctx; n.group_starts = to->group_starts; n.shared = to->shared;
    if (a.status) n.status = to->status;
  }
  __syncthreads();
  if (a.G && !__syncthreads_and(beam::ascends(n.group_starts, a.G, a.S, tid, threads) && beam::ascends(n.starts, a.S, a.T, tid, threads))) n.G = 0;
  return n;
}

// ---- items: a part's key head and a block of its rows.  Parts of up to 32 rows go to narrow CTAs, to teams of 1 or 2 warps with 16 rows each; the others (team 0) to wide ones, 256 rows
// a block.  An item's keys come in units: pages, or steps of a wide CTA, which has two tiles of 128 scores at once: those of two row tiles and 128 keys where there are more than 128 rows, else of
// one row tile and 256 keys.
__device__ __forceinline__ int team_of(int rows) { return rows <= kTile16 ? 1 : rows <= kNarrow ? 2 : 0; }
struct Items {
  int team, group, bt, bt_log;      // bt: tokens of a block, a power of two
  __device__ __forceinline__ Items(int team, int group) : team(team), group(group), bt_log((team ? 4 + (team > 1) : 8) - (group > 1) - (group > 2) - (group > 4)) { bt = 1 << bt_log; }
  // whether a part of so many rows is this team's
  __device__ __forceinline__ bool has(const Part& p) const { return p.rows && team_of(p.rows * group) == team; }
  // part u, without rows where it is another team's
  __device__ __forceinline__ Part part(const Lengths& n, int u) const {
    Part p = beam::part_of(n, u);
    if (!has(p)) p.rows = 0;
    return p;
  }
  __device__ __forceinline__ int unit_log(int tokens) const { return team ? 4 : 2 * tokens > bt ? 7 : 8; }
  __device__ __forceinline__ int end_of(const Part& p, int block) const { return p.all ? p.k1 : p.ctx + min(p.rows, (block + 1) << bt_log); }
  __device__ __forceinline__ int units_of(const Part& p, int block) const {
    const int log = unit_log(min(bt, p.rows - (block << bt_log)));
    return (end_of(p, block) - p.k0 + (1 << log) - 1) >> log;
  }
  __device__ __forceinline__ int blocks_of(const Part& p) const { return (p.rows + bt - 1) >> bt_log; }
  __device__ __forceinline__ int head_cost(const Part& p) const {
    const int blocks = blocks_of(p);
    if (blocks <= 1) return blocks ? units_of(p, 0) + tree::kItem : 0;
    int n = units_of(p, blocks - 1) + tree::kItem;      // (the last block may be of the other unit)
    if (p.all) return n + (blocks - 1) * (units_of(p, 0) + tree::kItem);
    for (int b = 0; b < blocks - 1; ++b) n += units_of(p, b) + tree::kItem;
    return n;
  }
};
struct Item {
  int u, kvh, block;
  Part p;
  int first, nb, k1, units;      // the block's tokens, the keys they may see
  __device__ __forceinline__ void fill(const Items& I) {
    first = block << I.bt_log;
    nb = min(I.bt, p.rows - first);
    k1 = I.end_of(p, block);
    units = I.units_of(p, block);
  }
  __device__ __forceinline__ void next(const Lengths& n, const Items& I, int kv_heads) {
    if (++block >= I.blocks_of(p)) {      // a head's blocks come one behind the other: CTAs side by side read the same pages
      block = 0;
      if (++kvh >= kv_heads) {
        kvh = 0;
        do p = I.part(n, ++u);
        while (p.rows == 0 && u + 1 < n.G + n.S);      // (a range's units are some part's, unless lengths change under the kernel)
      }
    }
    fill(I);
  }
};

// What the items of each kind cost, in front of a thread's share of the step's parts and in all.  Kinds: teams of 1 and 2 warps, and wide CTAs.
template <int kKinds>
struct Costs {
  int per;      // parts of a share
  int before[kKinds], all[kKinds];
};
__device__ __forceinline__ int kind_team(int kind) { return kind == 2 ? 0 : 1 << kind; }
// ... with one barrier
template <int kThreads, int kKinds>
__device__ __forceinline__ void find_costs(const Lengths& n, int kv_heads, int group, int (*sums)[4], Costs<kKinds>* c) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int U = n.G + n.S, per = (U + kThreads - 1) / kThreads, end = min(U, (tid + 1) * per);
  c->per = per;
  int own[kKinds];
#pragma unroll
  for (int i = 0; i < kKinds; ++i) own[i] = 0;
  for (int u = tid * per; u < end; ++u) {
    const Part p = beam::part_of(n, u);
    const int team = team_of(p.rows * group), cost = p.rows ? Items(team, group).head_cost(p) * kv_heads : 0;
#pragma unroll
    for (int i = 0; i < kKinds; ++i) own[i] += team == kind_team(i) ? cost : 0;
  }
#pragma unroll
  for (int i = 0; i < kKinds; ++i) {
    int x = own[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp][i] = x;
    c->before[i] = x - own[i];
    c->all[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w)
#pragma unroll
    for (int i = 0; i < kKinds; ++i) {
      const int x = sums[w][i];
      if (w < warp) c->before[i] += x;
      c->all[i] += x;
    }
}

// The ranges of CTA `cta` of the `ctas` that a kind has, of `streams` at most each: all items' units are cut into as many as there are, none with less than `least` units, and every CTA has as many
// of them, side by side, where there are fewer: the memory of all SMs is wanted.  A thread each looks for the share of parts that an end lies in.  first: the CTA's first range; range [count][2],
// where [count][4]: part, key head, block, and the first unit of the item that a range begins in.  Returns all ranges; to be followed by a barrier.
template <int kThreads, int kKinds>
__device__ __forceinline__ tree::Ranges find_ranges(const Lengths& n, const Items& I, const Costs<kKinds>& c, int kind, int kv_heads, int cta, int ctas, int streams, int least, int* shares, int* first,
                                                    int* count, int (*range)[2], int (*where)[4]) {
  const int tid = threadIdx.x;
  int N = c.all[0], before = c.before[0];
#pragma unroll
  for (int i = 1; i < kKinds; ++i)
    if (i == kind) N = c.all[i], before = c.before[i];
  shares[tid] = before;
  tree::Ranges ranges = tree::ranges_of(N, max(1, min(ctas * streams, N / least)));
  if (N == 0) ranges.n = 0;
  const int per = (ranges.n + ctas - 1) / ctas;
  *first = cta * per;
  *count = max(0, min(per, ranges.n - *first));
  __syncthreads();
  const int e = tid >> 1, end = tid & 1, r = *first + e + end;
  if (e < *count) {
    int at = N;      // behind the last item
    if (r < ranges.n) {
      const int b = ranges.at(r), share = tree::last_at_most(shares, kThreads - 1, b);      // the last share that begins there or in front of it: one with items
      int u = share * c.per, g0 = shares[share], head;
      Part p;
      for (;; ++u) {
        p = I.part(n, u);
        head = I.head_cost(p);
        if (b < g0 + head * kv_heads || u + 1 >= n.G + n.S) break;
        g0 += head * kv_heads;
      }
      const int kvh = head ? min((b - g0) / head, kv_heads - 1) : 0;
      g0 += kvh * head;
      int block = 0, units = I.units_of(p, 0);
      while (b >= g0 + units + tree::kItem && block + 1 < I.blocks_of(p)) g0 += units + tree::kItem, units = I.units_of(p, ++block);
      at = tree::snapped(b, g0, units, ranges.snap);
      if (!end) where[e][0] = u, where[e][1] = kvh, where[e][2] = block, where[e][3] = g0;
    }
    range[e][end] = at;
  }
  return ranges;
}

}  // namespace shared_attn

}  // namespace b200
