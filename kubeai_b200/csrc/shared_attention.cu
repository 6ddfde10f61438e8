// Attention over the paged cache for groups of requests whose first pages are the same.
//
//   out_t = sum_j softmax_j(scale q_t . k_j) v_j    over the shared keys j < P, once for all rows of a group, and the request's own j >= P up to the row itself
//
// Softmax over two sets of keys is a weighted sum of softmaxes over each, so the rows of a group meet the shared pages in an item of their own and every request's rows the pages behind
// them in another, and the two are joined by their maxima and sums.
// An item is a key head and rows (row = token * group + head) with a range of keys.  Parts of up to 32 rows go to narrow CTAs, whose teams of 1 or 2 warps have 16 rows a warp; the others to wide
// ones (shared_attention_wide.cuh).  One launch has both: its CTAs are shared out to the kinds by their work, and all items' keys of a kind, one behind the other, are cut into as many equal ranges as
// it has teams or CTAs.  (In two launches, either waits for the other's SMs: 16 x 8 beams took 79 us so and 72.5 in one, 128 rows behind 2048 tokens 62 and 50.)
// A team walks its range without a gap: its first warp loads pages ahead by TMA (128-byte swizzle) into the team's ring, over an item's end, and all multiply with mma.sync: row tiles of 16 leave the
// tensor cores idle in any form, and memory is what bounds this.
// An item that a range's end cuts leaves unnormalised rows in the workspace, as every item does that shares its rows with another; a second kernel joins them in a fixed order.
// 16 x 8 beams behind up to 4001 tokens, 273 MB: 67.4 us, of which the join has 6 and the first kernel 61, 4.5 TB/s (pages of random places by TMA reach 5.8 with nothing else to do): the last team ends 15 %
// behind the mean one, as what each gets of the memory differs.  128 rows behind 2048 tokens, 144 MB: 50.5.  64 x 8 beams behind up to 450, 173 MB: 62.7; three warps a scheduler wait on their own chains
// (products, maxima, exponentials, products), at two of three a page's time, and 168 registers leave no more.  What the loads know of their place lies in shared memory: in registers it spilled others (72).
// 1 x 4 beams behind 450: 13.8, a chain of lengths, costs, ranges (4 us of them, most of it instructions' first way from memory), page table, four pages, the rows' way out and the join.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "gemm.h"
#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "shared_attention.cuh"
#include "shared_attention_wide.cuh"

namespace b200 {
namespace {

using namespace shared_attn;
constexpr int kPageBytes = 2 * 16 * kD * 2;      // bytes of a page's keys and values of a head
constexpr int kDepth = 2, kItems = 4, kLeast = 4;      // kDepth: pages a warp on their way, 16 KB, 192 of an SM; kItems: items a warp that those may lie in, and one; kLeast: pages of a range
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kAtOnce = 4, kJoinPlaces = 4;      // kAtOnce: parts of a row on their way; kJoinPlaces: CTAs an SM, one wave, up to which more warps have a row's head
// The two forms of the kernel: with CTAs that may be wide, one an SM; and without, three an SM, which begin sooner: 1 x 4 beams behind 450 tokens took 16.3 us so, and 18.1 in the other form.
template <bool kWide>
struct Form {
  static constexpr int kThreads = kWide ? wide::kThreads : 128, kWarps = kThreads / 32, kPlaces = wide::kThreads / kThreads, kKinds = kWide ? 3 : 2;
  static constexpr int kRings = 1024 + kWarps * kDepth * kPageBytes, kSmem = kWide ? std::max(kRings, wide::kSmem) : kRings;
};
// What a page of each team, and a step of a wide CTA, take of an SM's time: by these the CTAs are shared out.  Teams of one next to wide CTAs: 128 rows behind 2048 tokens 24 52.8 us, 26 50.9, 28 51.2, 30 50.4;
// 64 groups of 48 rows behind 450 101.1, 101.1, 102.9, 104.2; 4 of 160 rows behind 8000 62.1, 61.7, 62.1, 63.5.  Teams of one and two: 16 x 8 beams 1.4 66.9, 1.6 67.3, 1.8 70.9, 64 x 8 behind 450 63.6, 62.7,
// 62.5.
__device__ constexpr float kShare[3] = {1.f, 1.6f, 26.f};

// An item's pages of a range, as the loads leave them for the products
struct Piece {
  int row0, rows, kvh;           // the first row of the step, rows (token * group + head)
  int key, pages;                // first key, pages
  int end, see;                  // keys behind the last, and behind the last that token 0 sees; token i sees i more
  int table;
  int whole, begins, own, joined, last;
  int parts;
};

template <int kWarps>
struct Narrow {
  uint64_t bars[2][kWarps * kDepth];
  Piece pieces[kWarps * kItems];
  Item items[kWarps];            // where the loads of each team are: kept here, as registers are wanted for the products
  int odd[kWarps * kItems];      // the last item of each piece's place with infinities or NaN among values that some row does not see
};
template <bool kWide> union Halves;
template <> union Halves<true> {
  Narrow<Form<true>::kWarps> narrow;
  wide::Shared wide;
  __device__ Halves() {}
};
template <> union Halves<false> {
  Narrow<Form<false>::kWarps> narrow;
  __device__ Halves() {}
};
static_assert(Form<true>::kSmem + sizeof(Halves<true>) + sizeof(Staged) + 3072 <= 227 * 1024, "");
static_assert(3 * (Form<false>::kSmem + sizeof(Halves<false>) + sizeof(Staged) + 2048) <= 228 * 1024, "");

template <bool kWide>
__global__ void __launch_bounds__(Form<kWide>::kThreads, Form<kWide>::kPlaces)
shared_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ b200_shared_attn_args a, const Sizes sizes, float scale_log2, int* error) {
  constexpr int kThreads = Form<kWide>::kThreads, kWarps = Form<kWide>::kWarps, kKinds = Form<kWide>::kKinds;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) Halves<kWide> both;
  __shared__ __align__(16) int sums[kWarps][4];
  __shared__ int shares[kThreads], s_range[kWarps][2], s_where[kWarps][4];
  __shared__ Staged staged;
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - smem_u32(smem_raw));
  const int warp = warp_number(), lane = threadIdx.x & 31, tid = threadIdx.x;
  const int group = a.q_heads / a.kv_heads, shift = __ffs(group) - 1;
  griddep_wait();
  griddep_launch();
  const Lengths n = lengths_of(a, &staged, tid, kThreads);
  // ---- which kind: CTAs by the work of each, one at least
  Costs<kKinds> costs;
  find_costs<kThreads>(n, a.kv_heads, group, sums, &costs);
  int kind = 0, first_cta = 0, its = gridDim.x, first, count;
  {
    float part[kKinds], all = 0.f;
#pragma unroll
    for (int i = 0; i < kKinds; ++i) part[i] = static_cast<float>(costs.all[i]) * kShare[i], all += part[i];
    const float each = gridDim.x / all;
    // rounded up, so that none is left far behind; what is left of the last kind, the wide CTAs where there are any: most of the work is theirs then, or they are as many as may be
    int left = gridDim.x, begin = 0;
#pragma unroll
    for (int k = 0; k < kKinds; ++k) {
      constexpr int kOrder[3] = {1, 0, 2};
      const int i = kOrder[k];
      int behind = 0;      // kinds behind it
#pragma unroll
      for (int j = k + 1; j < kKinds; ++j) behind += costs.all[kOrder[j]] > 0;
      int count = costs.all[i] == 0 ? 0 : behind == 0 ? left : max(1, min(left - behind, static_cast<int>(ceilf(part[i] * each))));
      if (i == 2) count = min(count, sizes.ctas);
      if (static_cast<int>(blockIdx.x) >= begin && static_cast<int>(blockIdx.x) < begin + count) kind = i, first_cta = begin, its = count;
      begin += count;
      left -= count;
    }
    if (static_cast<int>(blockIdx.x) >= begin) return;      // nothing that it might have
  }
  // (one look for the ranges of either half: what comes once costs its instructions' way from memory)
  const int cta = blockIdx.x - first_cta, team = kind_team(kind), streams = team ? kWarps >> kind : 1;
  static_assert(kLeast == wide::kLeast, "");
  const Items I(team, group);
  const tree::Ranges ranges = find_ranges<kThreads>(n, I, costs, kind, a.kv_heads, cta, its, streams, kLeast, shares, &first, &count, s_range, s_where);
  if constexpr (kWide) {
    if (!team) {
      if (count) wide::walk(tm_q, tm_kv, a, sizes, scale_log2, error, smem, both.wide, n, ranges, cta, s_range[0], s_where);
      return;
    }
  }
  if (tid < kWarps * kItems) both.narrow.odd[tid] = -1;
  const int stream = warp >> kind, member = warp & (team - 1);
  static_assert(kDepth == 2, "");
  const int depth = kDepth * team, depth_log = kind + 1, cap = kItems * team;
  const uint32_t ring = sbase + stream * depth * kPageBytes, full0 = smem_u32(both.narrow.bars[0] + stream * depth), empty0 = smem_u32(both.narrow.bars[1] + stream * depth);
  Piece* pieces = both.narrow.pieces + stream * cap;
  volatile int* odd_item = both.narrow.odd + stream * cap;
  if (lane == 0 && member == 0) {
    for (int s = 0; s < depth; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, team);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tm_kv);
  }
  __syncthreads();
  const int gs = first + stream;      // the team's range
  const int left = stream < count ? s_range[stream][1] - s_range[stream][0] : 0;
  if (left <= 0) return;
  const Space space = space_of(a, sizes);
  const int slot = (first_cta * kWarps + gs * team) * 2;      // of 16 rows: the range's first item, a team's tiles behind it the last

  // ---- loads (the team's first warp): item, its first page here, the range's cost to go
  Item& it = both.narrow.items[stream];
  if (member == 0 && lane == 0) {
    it.u = s_where[stream][0]; it.kvh = s_where[stream][1]; it.block = s_where[stream][2];
    it.p = I.part(n, it.u);
    it.fill(I);
  }
  auto go_on = [&] {
    __syncwarp();
    if (lane == 0) it.next(n, I, a.kv_heads);
    __syncwarp();
  };
  __syncwarp();
  int t0 = max(0, s_range[stream][0] - s_where[stream][3] - tree::kItem), rest = left;
  if (member == 0 && t0 == it.units) {              // the range begins where the item in front of it ends
    t0 = 0;
    go_on();
  }
  bool more = true, ok = true;
  int take = 0, at = 0, items = 0, issued = 0, mine = 0, next = 0;      // the item's pages here, the page that is next; items so far; pages so far
  const bool one = elect_one();
  // the first row of a page's keys; a page that the cache does not have lies behind its last row, where a load finds zeros
  auto look_up = [&](int p) {
    const int page = p < t0 + take ? a.block_tables[static_cast<size_t>(it.p.table) * a.ld_tables + it.p.k0 / 16 + p] : -1;
    return ((page >= 0 && page < a.num_pages ? page : static_cast<int>(a.num_pages)) * 2 * a.kv_heads + it.kvh) * 16;
  };
  auto begin = [&] {
    take = tree::take_of(t0, it.units, &rest);
    at = 0;
    mine = look_up(t0 + lane);
    next = look_up(t0 + 32 + lane);
    if (lane == 0) {
      const bool whole = t0 == 0 && take == it.units;
      Piece x;
      x.row0 = it.p.row0 + it.first;
      x.rows = it.nb * group;
      x.kvh = it.kvh;
      x.key = it.p.k0 + 16 * t0;
      x.pages = take;
      x.end = it.k1;
      x.see = it.p.all ? it.k1 : it.p.ctx + it.first + 1;
      x.table = it.p.table;
      x.whole = whole;
      x.begins = t0 == 0;
      x.own = !it.p.all;
      x.joined = it.p.k0 > 0;
      x.parts = whole ? 0 : t0 == 0 ? ranges.parts(gs, s_range[stream][1] - take, it.units) : 0;
      x.last = rest <= 0;
      pieces[items & (cap - 1)] = x;
    }
    ++items;
    __syncwarp();
  };
  // the next page of the range, into the place of the one that was used last
  auto load = [&] {
    if (!more) return;
    if (at == take) {
      if (rest <= 0) { more = false; return; }
      t0 = 0;
      go_on();
      begin();
    } else if (at && at % 32 == 0) {
      mine = next;
      next = look_up(t0 + at + 32 + lane);
    }
    const int row = __shfl_sync(0xffffffffu, mine, at & 31), st = issued & (depth - 1);
    if (team > 1 && !(ok = warp_wait(empty0 + 8 * st, ((issued >> depth_log) & 1) ^ 1u))) return;      // all warps of the team have read what lay there
    const uint32_t full = full0 + 8 * st, dst = ring + st * kPageBytes;
    if (one) {
      mbar_arrive_expect_tx(full, kPageBytes);
      tma_load_2d(dst, &tm_kv, full, 0, row, kEvictNormal);
      tma_load_2d(dst + 2048, &tm_kv, full, 64, row, kEvictNormal);
      tma_load_2d(dst + 4096, &tm_kv, full, 0, row + 16 * a.kv_heads, kEvictNormal);
      tma_load_2d(dst + 6144, &tm_kv, full, 64, row + 16 * a.kv_heads, kEvictNormal);
    }
    __syncwarp();
    ++at;
    ++issued;
  };
  if (member == 0) {
    begin();
    for (int k = 0; k < depth; ++k) load();
  }

  // ---- products: this thread has rows g and g + 8
  const int g = lane >> 2, q2 = (lane & 3) * 2, rr = lane & 7, tile = lane >> 3;
  const uint32_t k_row = rr + (tile >> 1) * 8, k_chunk = tile & 1, v_row = rr + (tile & 1) * 8, v_chunk = tile >> 1;
  int used = 0;
  for (int item = 0; ok; ++item) {
    if (team > 1 && !(ok = warp_wait(full0 + 8 * (used & (depth - 1)), (used >> depth_log) & 1))) break;      // the item's first page, and in front of it the piece, which a warp alone has written itself
    const Piece& x = pieces[item & (cap - 1)];      // (its place is used again some items on)
    const int rows = x.rows, first_key = x.key, pages_here = x.pages, see = x.see, end = x.end;
    const int r0 = 16 * member;
    const bool some = r0 < rows;      // this warp has rows
    // queries: rows nobody owns are zeros
    uint32_t qa[8][4];
    const bf16* q = static_cast<const bf16*>(a.q) + x.kvh * group * kD + q2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + g + 8 * h;
      const bf16* from = q + static_cast<size_t>(x.row0 + (r >> shift)) * a.ldq + (r & (group - 1)) * kD;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        qa[ks][h] = r < rows ? *reinterpret_cast<const uint32_t*>(from + ks * 16) : 0u;
        qa[ks][2 + h] = r < rows ? *reinterpret_cast<const uint32_t*>(from + ks * 16 + 8) : 0u;
      }
    }
    float o[16][4];
#pragma unroll
    for (int d = 0; d < 16; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[d][c] = 0.f;
    float ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // what the weights are relative to, in units of log 2; this thread's part of their sum
    const int limit[2] = {min(see + ((r0 + g) >> shift), end), min(see + ((r0 + g + 8) >> shift), end)};
    for (int j = 0; j < pages_here; ++j, ++used) {
      const int st = used & (depth - 1), key0 = first_key + 16 * j;
      if (!(ok = warp_wait(full0 + 8 * st, (used >> depth_log) & 1))) break;
      const uint32_t ks_ = ring + st * kPageBytes, vs_ = ks_ + 4096;
      if (some) {
      if (key0 + 16 > see) {
        // what must not meet a weight of zero: values behind the last key, and infinities and NaN among values that some row does not see, which those that do add at the end
        uint4* v = reinterpret_cast<uint4*>(smem + (vs_ - sbase));
        for (int e = lane; e < 256; e += 32) {
          bool found;
          const int key = key0 + ((e & 127) >> 3);      // (a row's pieces in some order)
          if (key < see) continue;
          uint4 w = v[e];
          if (key >= end) w = make_uint4(0, 0, 0, 0);
          else {
            const uint4 was = w;
            w = make_uint4(without_odd(w.x), without_odd(w.y), without_odd(w.z), without_odd(w.w));
            found = w.x != was.x || w.y != was.y || w.z != was.z || w.w != was.w;
            if (found) {      // ahead of what another warp of the team may find without them
              odd_item[item & (cap - 1)] = item;
              __threadfence_block();
            }
          }
          v[e] = w;
        }
        fence_proxy_async();
        __syncwarp();
      }
      float s[2][4];
#pragma unroll
      for (int c = 0; c < 4; ++c) s[0][c] = s[1][c] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(ks_ + (ks >> 2) * 2048 + k_row * 128 + ((((ks & 3) * 2 + k_chunk) ^ (k_row & 7)) << 4), b0, b1, b2, b3);
        mma_bf16_16816(s[0], qa[ks], b0, b1);
        mma_bf16_16816(s[1], qa[ks], b2, b3);
      }
      if (key0 + 16 > see) {
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (key0 + nb * 8 + q2 + (c & 1) >= limit[c >> 1]) s[nb][c] = -INFINITY;
      }
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * scale_log2;
        alpha[h] = 1.f;
        if (top > ref[h]) {
          alpha[h] = exp2_ftz(ref[h] - top);
          ref[h] = top;
        }
      }
      uint32_t pa[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mu = ref[h] == -INFINITY ? 0.f : ref[h];
        float ps = 0.f;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          const uint32_t w = pack_bf16x2(exp2_ftz(fmaf(s[nb][2 * h], scale_log2, -mu)), exp2_ftz(fmaf(s[nb][2 * h + 1], scale_log2, -mu)));
          // the sum is that of the rounded weights: where one weight outweighs the others, its rounding cancels
          ps += __uint_as_float(w << 16) + __uint_as_float(w & 0xffff0000u);
          pa[2 * nb + h] = w;
        }
        l[h] = l[h] * alpha[h] + ps;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int d = 0; d < 16; ++d)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[d][c] *= alpha[c >> 1];
      }
#pragma unroll
      for (int dp = 0; dp < 8; ++dp) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(vs_ + (dp >> 2) * 2048 + v_row * 128 + ((((dp & 3) * 2 + v_chunk) ^ (v_row & 7)) << 4), b0, b1, b2, b3);
        mma_bf16_16816(o[2 * dp], pa, b0, b1);
        mma_bf16_16816(o[2 * dp + 1], pa, b2, b3);
      }
      }
      __syncwarp();      // all have read the page
      if (team > 1 && lane == 0) mbar_arrive(empty0 + 8 * st);
      if (member == 0) load();
      if (!ok) break;
    }
    if (!ok) break;
    // ---- the item's rows
    __threadfence_block();
    if (some && odd_item[item & (cap - 1)] == item) {
      for (int p = max(x.see, x.key); p < min(x.end, x.key + 16 * x.pages); ++p) {
        const long long row = tree::cache_row(a.block_tables + static_cast<size_t>(x.table) * a.ld_tables, p, a.num_pages);
        if (row < 0) continue;
        const bf16* value = static_cast<const bf16*>(a.kv_layer) + ((((row >> 4) * 2 + 1) * a.kv_heads + x.kvh) * 16 + (row & 15)) * kD + q2;
#pragma unroll
        for (int d = 0; d < 16; ++d)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float y = __bfloat162float(value[d * 8 + (c & 1)]);
            if (!isfinite(y) && p < limit[c >> 1]) o[d][c] += y;
          }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    if (x.begins && member == 0)
      for (int i = lane; i < x.rows >> shift; i += 32)
        space.places[(static_cast<size_t>(x.own) * a.T + x.row0 + i) * a.kv_heads + x.kvh] = {slot + team, x.parts, i << shift, kTeam * team + (x.joined ? kJoined : 0)};
    const bool last = x.whole && x.own && !x.joined;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + g + 8 * h;
      if (r >= x.rows) continue;
      const size_t t = static_cast<size_t>(x.row0 + (r >> shift));
      const int head = x.kvh * group + (r & (group - 1));
      if (last) {
        const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
        bf16* out = static_cast<bf16*>(a.out) + t * a.ldo + head * kD + q2;
#pragma unroll
        for (int d = 0; d < 16; ++d) *reinterpret_cast<uint32_t*>(out + d * 8) = pack_bf16x2(o[d][2 * h] * inv, o[d][2 * h + 1] * inv);
      } else {
        float* out = x.whole ? space.rows + ((static_cast<size_t>(x.own) * a.T + t) * a.q_heads + head) * kLd : space.narrow + (static_cast<size_t>(slot + (x.begins ? team : 0)) * kTile16 + r) * kLd;
#pragma unroll
        for (int d = 0; d < 16; ++d) *reinterpret_cast<float2*>(out + d * 8 + q2) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(out + kD) = make_float2(ref[h], l[h]);
      }
    }
    if (x.last) break;
  }
  // the copies in flight land before the CTA ends, also where it gives up
  for (int k = used; k < issued; ++k) warp_wait(full0 + 8 * (k & (depth - 1)), (k >> depth_log) & 1);
  if (!ok) *reinterpret_cast<volatile int*>(error) = 1;
}

// Bound by its dependent trips: places, maxima with four parts' outputs, further ones; six or eight parts at a time cost more registers and instructions than they save trips (16 x 8 beams 74 and 74.7 us).
// A row: sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p over the parts, in order, four dimensions a lane; a lane has the maximum, sum and weight of one part in 32.
struct Joined {
  float m, sum;
  float4 y;
};
template <typename At>
__device__ __forceinline__ Joined join_parts(int parts, At part, int lane) {
  Joined j = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int p0 = 0; p0 < parts; p0 += 32) {
    const int count = min(32, parts - p0);
    const float* mine = part(p0 + min(lane, count - 1));
    float4 x[kAtOnce];
    auto load = [&](int k0) {
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), (k0 + k) & 31));
        if (k0 + k < count) x[k] = *reinterpret_cast<const float4*>(from + lane * 4);
      }
    };
    const float2 st = lane < count ? *reinterpret_cast<const float2*>(mine + kD) : make_float2(-INFINITY, 0.f);
    load(0);
    float top = fmaxf(j.m, st.x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top, old = exp2f(j.m - base), w = exp2f(st.x - base);
    j.m = top;
    float l = w == 0.f && st.y == st.y ? 0.f : st.y * w;
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    j.sum = j.sum * old + l;
    j.y = make_float4(j.y.x * old, j.y.y * old, j.y.z * old, j.y.w * old);
    for (int k0 = 0; k0 < count; k0 += kAtOnce) {
      if (k0) load(k0);
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float wk = __shfl_sync(0xffffffffu, w, (k0 + k) & 31);
        if (k0 + k < count && wk != 0.f) j.y = make_float4(fmaf(x[k].x, wk, j.y.x), fmaf(x[k].y, wk, j.y.y), fmaf(x[k].z, wk, j.y.z), fmaf(x[k].w, wk, j.y.w));
      }
    }
  }
  return j;
}

// Whether all parts of a place lie in the workspace: not so where a wait ran out in front of it and it was not written
__device__ __forceinline__ bool in_bounds(const Place& p, const Sizes& sizes, int group) {
  if (p.parts == 0) return true;
  const int team = p.flags / kTeam, behind = max(1, team);
  const long long first = p.slot, last = first - behind + 2ll * behind * (p.parts - 1), slots = 2ll * (team ? sizes.warps : sizes.ctas) - behind;
  return p.parts > 0 && p.flags >= 0 && team <= 2 && first >= behind && first <= slots && last <= slots && p.row >= 0 && p.row <= (team ? team * kTile16 : kWideRows) - group;
}

// kWarps have a head of a row, and every kWarps-th of its parts each: as many as leave one wave of CTAs.  1 x 4 beams behind 1500 tokens 20 us -> 15.3, behind 4000 31 -> 17.7 (14.3 and
// 16.8 since); in two waves 128 rows behind 2048 tokens took 52.9, and 50 in one.
template <int kWarps>
__global__ void __launch_bounds__(kJoinThreads)
shared_attn_join_kernel(const __grid_constant__ b200_shared_attn_args a, const Sizes sizes) {
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, head = (blockIdx.y * kJoinWarps + warp) / kWarps, member = warp % kWarps;
  __shared__ Joined joined[kWarps > 1 ? kJoinWarps : 1][32];
  // the lengths were there before the kernel in front of this one let it in
  griddep_launch();
  // whether some request has the row: where starts ascend the last one that begins there or in front of it, found among 65536 in two looks of a value a thread; else any (16384 requests: 1356 us for looking
  // at all of them for every row)
  const int apart = (a.S + kJoinThreads - 1) / kJoinThreads;
  const int near = max(0, __syncthreads_count(tid * apart < a.S && a.starts[tid * apart] <= t) - 1) * apart;
  const int at = apart == 1 ? near : near + max(0, __syncthreads_count(tid < apart && near + tid < a.S && a.starts[near + tid] <= t) - 1);
  auto has = [&](int s) {
    const tree::Request r = tree::request_of(a.starts, a.ctx, s, a.T, a.max_blocks, a.max_rows, a.status);
    return t >= r.row0 && t < r.row0 + r.rows;
  };
  bool mine = has(at);
  if (!mine) {
    for (int s = tid; s < a.S && !mine; s += kJoinThreads) mine = has(s);
    mine = __syncthreads_or(mine);
  }
  griddep_wait();
  const Space space = space_of(a, sizes);
  const int group = a.q_heads / a.kv_heads, kvh = min(head, a.q_heads - 1) / group;
  // (what lies there counts where some request has the row)
  const Place shared = space.places[static_cast<size_t>(t) * a.kv_heads + kvh], own = space.places[(static_cast<size_t>(a.T) + t) * a.kv_heads + kvh];
  if (head >= a.q_heads) return;
  uint2* out = reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + static_cast<size_t>(t) * a.ldo + head * kD) + lane;
  if (!mine) {
    if (a.zero_rest && !member) *out = make_uint2(0, 0);
    return;
  }
  if (!own.parts && !(own.flags & kJoined)) return;      // written already
  if (!in_bounds(own, sizes, group) || (own.flags & kJoined && !in_bounds(shared, sizes, group))) return;
  const int n_own = max(1, own.parts), n_all = n_own + (own.flags & kJoined ? max(1, shared.parts) : 0);
  // an item's beginning lies in its range's second slot, each other part in its range's first
  auto part = [&](int p) -> const float* {
    const bool first = p < n_own;
    const int k = first ? p : p - n_own, parts = first ? own.parts : shared.parts, slot = first ? own.slot : shared.slot, row = first ? own.row : shared.row;
    if (!parts) return space.rows + ((static_cast<size_t>(first) * a.T + t) * a.q_heads + head) * kLd;
    const int team = (first ? own.flags : shared.flags) / kTeam, behind = max(1, team);      // from a range's second slot to its first, and half of what lies between two ranges
    return (team ? space.narrow : space.wide) + (static_cast<size_t>(k ? slot - behind + 2 * behind * k : slot) * (team ? kTile16 : kWideRows) + row + head % group) * kLd;
  };
  Joined j;
  if constexpr (kWarps > 1) {
    joined[warp][lane] = join_parts((n_all + kWarps - 1 - member) / kWarps, [&](int p) { return part(p * kWarps + member); }, lane);
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / kWarps), "n"(kWarps * 32) : "memory");      // (a head's warps take every way together)
    if (member) return;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, joined[warp + w][lane].m);
    j = {m, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const Joined x = joined[warp + w][lane];
      const float f = exp2f(x.m - base);
      if (f == 0.f && x.sum == x.sum) continue;
      j.sum += x.sum * f;
      j.y = make_float4(fmaf(x.y.x, f, j.y.x), fmaf(x.y.y, f, j.y.y), fmaf(x.y.z, f, j.y.z), fmaf(x.y.w, f, j.y.w));
    }
  } else
    j = join_parts(n_all, part, lane);
  const float inv = j.sum == 0.f ? 0.f : 1.f / j.sum;
  *out = make_uint2(pack_bf16x2(j.y.x * inv, j.y.y * inv), pack_bf16x2(j.y.z * inv, j.y.w * inv));
}

// Where only the order of `starts` keeps what all parts cost within 32 bits: a copy, in which nobody has rows if they do not ascend
__global__ void __launch_bounds__(1024)
ordered_starts_kernel(const int* starts, int S, int T, int* to) {
  griddep_enter();
  const bool ordered = __syncthreads_and(beam::ascends(starts, S, T, threadIdx.x, 1024));
  for (int s = threadIdx.x; s <= S; s += 1024) to[s] = ordered ? starts[s] : 0;
}

}  // namespace

// How many CTAs may be wide: none where no part can have so many rows, else as many as there are SMs, or as the most work that the call may have feeds
static int wide_ctas(const b200_shared_attn_args& a) {
  const long long group = a.q_heads / a.kv_heads, T = a.T, most = std::min<long long>(a.max_rows, T);
  const bool shared = a.G && T * group > kNarrow, own = most * group > kNarrow;
  if (!shared && !own) return 0;
  const long long seen = std::min<long long>(a.max_ctx ? a.max_ctx : INT_MAX, a.max_blocks * static_cast<long long>(tree::kPage)) + most;
  const long long items = ((shared ? (T * group + kWideRows - 1) / kWideRows + a.G : 0) + (own ? (most * group + kWideRows - 1) / kWideRows * a.S : 0)) * a.kv_heads;
  return static_cast<int>(std::min<long long>(sm_count(), std::max<long long>(1, items * ((seen + wide::kKeys - 1) / wide::kKeys + tree::kItem) / wide::kLeast)));
}

static Sizes sizes_of(const b200_shared_attn_args& a) { return {sm_count() * Form<true>::kWarps, wide_ctas(a)}; }

// The copy of `starts`, behind everything else
static int64_t starts_bytes(const b200_shared_attn_args& a) { return beam::costs_fit(a, false) ? 0 : (a.S + 4ll) / 4 * 16; }

int64_t shared_attention_workspace(const b200_shared_attn_args& a) {
  const Sizes n = sizes_of(a);
  const int64_t T = a.T;
  return 2 * T * a.kv_heads * static_cast<int64_t>(sizeof(Place)) +
         (2ll * n.warps * kTile16 + 2ll * n.ctas * kWideRows + (a.G ? 2 * T * a.q_heads : 0)) * kLd * static_cast<int64_t>(sizeof(float)) + starts_bytes(a);
}

int paged_attention_shared(const b200_shared_attn_args& args, int* error, cudaStream_t st) {
  b200_shared_attn_args a = args;
  const Sizes sizes = sizes_of(a);
  if (const int64_t bytes = starts_bytes(a)) {
    int* starts = reinterpret_cast<int*>(static_cast<uint8_t*>(a.workspace) + shared_attention_workspace(a) - bytes);
    launch_pdl(ordered_starts_kernel, dim3(1), dim3(1024), 0, st, a.starts, a.S, a.T, starts);
    if (cudaGetLastError() != cudaSuccess) return -2;
    a.starts = starts;
  }
  const int group = a.q_heads / a.kv_heads;
  CUtensorMap tm_kv, tm_q;
  if (int rc = tmap_encode_bf16_2d(&tm_kv, a.kv_layer, static_cast<uint64_t>(a.num_pages) * 2 * a.kv_heads * 16, kD, kD, 16, 64, 1)) return rc;
  tm_q = tm_kv;
  if (sizes.ctas)
    if (int rc = tmap_encode_bf16_3d(&tm_q, a.q, kD, a.q_heads, a.T, kD, a.ldq, 64, group, wide::kTileRows / group)) return rc;
  auto launch = [&](auto kernel, auto form, std::atomic<unsigned long long>* attr_done) {
    using F = decltype(form);
    if (!ensure_dynamic_smem(kernel, F::kSmem, attr_done)) return -3;
    launch_pdl(kernel, dim3(sizes.warps / F::kWarps), dim3(F::kThreads), F::kSmem, st, tm_q, tm_kv, a, sizes, a.scale * 1.4426950408889634f, error);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
  };
  static std::atomic<unsigned long long> wide_done{0}, narrow_done{0};
  if (int rc = sizes.ctas ? launch(shared_attn_kernel<true>, Form<true>{}, &wide_done) : launch(shared_attn_kernel<false>, Form<false>{}, &narrow_done)) return rc;
  auto join = [&](auto kernel, int warps) { launch_pdl(kernel, dim3(a.T, (a.q_heads * warps + kJoinWarps - 1) / kJoinWarps), dim3(kJoinThreads), 0, st, a, sizes); };
  const long long most = static_cast<long long>(kJoinPlaces) * sm_count() * kJoinWarps, heads = static_cast<long long>(a.T) * a.q_heads;
  if (heads * 8 <= most) join(shared_attn_join_kernel<8>, 8);
  else if (heads * 4 <= most) join(shared_attn_join_kernel<4>, 4);
  else if (heads * 2 <= most) join(shared_attn_join_kernel<2>, 2);
  else join(shared_attn_join_kernel<1>, 1);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
