// Attention of the rows of drafted trees over the paged cache, on the 5th-generation tensor cores.
//
//   out_t = sum_j softmax_j(scale q_t . k_j) v_j   over j < ctx and those j = ctx + i whose bit i the row's mask has
//
// A request's rows share all keys but the last few, so what counts is that K and V pass once for all rows of a key head and that nothing stops the stream
// of pages.  An item is a request's key head and up to 128 of its rows (row = token * group + head); its keys come in tiles of 64.  All items' tiles one behind the
// other are cut into as many equal ranges as the SMs have places for CTAs, two each, and a CTA walks its range without a gap:
//   two warps look pages up (32 of the table at a time, the next ones ahead) and load by TMA, 128-byte swizzle, into rings, one queries and keys, one values;
//   two warps issue tcgen05.mma, one S = Q K^T (M = 128, N = 64, two buffers), one O += P V (M = 128, N = 128, P in TMEM over its scores): a wait that is over
//   costs its warp 100 cycles all the same, and one warp for both took 1500 a tile of which the tensor cores need 640;
//   four warps (thread = row) do the softmax in fp32, base 2; a warp whose rows nobody owns only keeps step.
// While one CTA of an SM ends an item, the other one keeps the memory busy.  (One CTA an SM with two softmax groups that took a row tile's keys in turn, or a row
// tile each, stopped for 3 us at each item: 64 x 2048 74.8 us.)  More than 128 rows: items side by side, which find each other's pages in L2.
// What bounds it: the chain of a tile through its softmax warps, 1850 to 2000 cycles from scores to weights (load and maximum, exponentials, weights back to tensor memory; 600 of
// them O's rescaling and the wait for the product ahead of it) and 400 more until the next scores are there, by two CTAs an SM; the exponentials' unit has work for 512 of a full
// tile.  64 requests of 2048 tokens, 32 heads on 8: 69 us, 320 MB, 4.7 TB/s (the second kernel's 6 us left out 5.1); two of 32001: 58 us, 4.6 TB/s; 48 of 1999 with 64
// rows, 256 rows of a key head: 93 us, exponentials' unit 27 % busy, tensor cores 32 %, issue slots 40 %.
// Weights are relative to the row's largest score so far, so the largest weight is exactly 1 and its rounding to bf16 costs nothing.  Relative to up to 2^8 times an older
// maximum, which saves most of the rescaling of O (63, 55 and 84 us), results were off by 1 to 13 % more (64 x 2048: 0.00232 of the output for 0.00222).
// The masks' bits are looked at only in tiles that reach behind the context.  There the products' warp also clears what must not meet a weight of zero:
// values behind the last key, and infinities and NaN among the drafts' values, which the rows that see them add at the end by themselves.
// An item that a range's end cuts leaves unnormalised rows in the workspace, which a second kernel joins in a fixed order: the same bits every time.
// Every wait has a limit; a CTA that gives up sets an error mark and still meets at the end.
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
#include "tree_step.h"

namespace b200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kD = 128, kRows = 128, kKeys = 64;
constexpr int kQSlab = kRows * 128, kSlab = kKeys * 128, kTile = 2 * kSlab;      // bytes: 64 columns of a row tile, of a key tile, a key tile
constexpr int kThreads = 256, kWarps = kThreads / 32, kPlaces = 2;                // kPlaces: CTAs of an SM
constexpr int kDepth = 2;                  // tiles of keys, and of values, on their way
constexpr int kLd = kD + 4;                // floats from row to row of the workspace: output, maximum, sum
constexpr int kJoinThreads = 256, kJoinPlaces = 3, kJoinAtOnce = 8, kFew = 4;      // kJoinPlaces: CTAs of an SM; kJoinAtOnce: parts on their way
constexpr int kWaitLimit = 1 << 22;

// shared memory: queries, keys, values, 2 KB a softmax warp for its way out, barriers
constexpr int kKeysAt = 2 * kQSlab, kValuesAt = kKeysAt + kDepth * kTile, kStageAt = kValuesAt + kDepth * kTile, kBars = kStageAt + 4 * 2048, kSmem = 1024 + kBars + 256;
static_assert(kPlaces * (kSmem + 1024 + 128) <= 228 * 1024, "");

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_limited(bar, parity, kWaitLimit)); }
// two bf16 without infinities and NaN
__device__ __forceinline__ uint32_t without_odd(uint32_t u) { return ((u & 0x7f80u) == 0x7f80u ? 0u : u & 0xffffu) | ((u & 0x7f800000u) == 0x7f800000u ? 0u : u & 0xffff0000u); }

// Which of the rows j .. j + 31 of its request row i sees (j may be negative: tokens of the context, all seen)
__device__ __forceinline__ uint32_t seen_bits(const int* mask, int words, int i, int rows, int j) {
  auto word = [&](int w) -> uint32_t {
    const int left = rows - 32 * w;
    const uint32_t inside = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
    if (!mask) return i - 32 * w >= 31 ? inside : i < 32 * w ? 0u : ((2u << (i - 32 * w)) - 1) & inside;
    return w < words ? static_cast<uint32_t>(mask[w]) & inside : 0u;
  };
  if (j <= -32) return ~0u;
  if (j < 0) return ~(~0u << -j) | word(0) << -j;
  return __funnelshift_r(word(j >> 5), word((j >> 5) + 1), j & 31);
}

__device__ __forceinline__ tree::Request request(const b200_tree_attn_args& a, int s) { return tree::request_of(a.starts, a.ctx, s, a.T, a.max_blocks, a.max_tree, a.status); }

// Of the rows that no request owns, and those of requests that are left out, every parts-th one becomes zeros (one block).
__device__ void zero_rest(const b200_tree_attn_args& a, int part, int parts) {
  bool ordered = true, all = true;      // rows one behind the other; of requests that are all served
  for (int s = threadIdx.x; s < a.S; s += blockDim.x) {
    const int begin = a.starts[s], end = a.starts[s + 1];
    ordered = ordered && begin >= 0 && begin <= end && end <= a.T;
    all = all && request(a, s).rows == end - begin;
  }
  ordered = __syncthreads_and(ordered);
  all = __syncthreads_and(all);
  const int from = ordered && a.S ? a.starts[0] : 0, to = ordered && a.S ? a.starts[a.S] : 0;
  for (int t = part; t < a.T; t += parts) {
    int end = 0;      // of the rows that are somebody's from t on
    if (ordered && t >= from && t < to) {
      if (all) end = to;
      else {
        const int s = tree::last_at_most(a.starts, a.S, t);
        if (request(a, s).rows) end = a.starts[s + 1];
      }
    }
    for (int s = 0; !ordered && s < a.S && !end; ++s) {
      const tree::Request r = request(a, s);
      if (t >= r.row0 && t < r.row0 + r.rows) end = t + 1;
    }
    if (end) { t += (end - 1 - t) / parts * parts; continue; }
    uint4* out = reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) + static_cast<size_t>(t) * a.ldo);
    for (int c = threadIdx.x; c < a.q_heads * (kD / 8); c += blockDim.x) out[c] = make_uint4(0, 0, 0, 0);
  }
}


// ---- items and ranges
struct Item {
  int s, kvh, block;              // request, key head, which of its blocks of rows
  tree::Request r;
  int first, nb, kv_end, tiles;   // the block's tokens, keys that they may see
};

__device__ __forceinline__ int block_tokens(const b200_tree_attn_args& a) { return kRows / (a.q_heads / a.kv_heads); }
__device__ __forceinline__ int tiles_of(const b200_tree_attn_args& a, const tree::Request& r, int bt, int block) {
  const int seen = a.masks ? r.rows : min(r.rows, (block + 1) * bt);
  return (r.ctx + seen + kKeys - 1) / kKeys;
}
__device__ __forceinline__ int blocks_of(const tree::Request& r, int bt) { return (r.rows + bt - 1) / bt; }
// what all blocks of a key head cost
__device__ __forceinline__ int head_cost(const b200_tree_attn_args& a, const tree::Request& r, int bt) {
  const int blocks = blocks_of(r, bt);
  if (a.masks || blocks <= 1) return blocks ? blocks * (tiles_of(a, r, bt, 0) + tree::kItem) : 0;
  int n = 0;
  for (int b = 0; b < blocks; ++b) n += tiles_of(a, r, bt, b) + tree::kItem;
  return n;
}
__device__ __forceinline__ void fill(const b200_tree_attn_args& a, int bt, Item* it) {
  it->first = it->block * bt;
  it->nb = min(bt, it->r.rows - it->first);
  it->kv_end = it->r.ctx + (a.masks ? it->r.rows : it->first + it->nb);
  it->tiles = tiles_of(a, it->r, bt, it->block);
}

// What a CTA leaves for the second kernel: the item that begins in its range and ends behind it, and in how many ranges it lies (0: no such item).
struct Cut {
  int row0, rows, kvh, parts;      // the item's first row of the step, rows (token * group + head)
};

// The workspace: a Cut and two parts' rows for every CTA
__host__ __device__ __forceinline__ float* rows_of(void* workspace, int ctas) { return reinterpret_cast<float*>(static_cast<Cut*>(workspace) + ctas); }

// Infinities and NaN of the drafts that a row sees, which stayed out of the products, to its dimensions c1 ..
__device__ __noinline__ void add_odd(const b200_tree_attn_args& a, const Item it, int t0, int take, int c1, int token, uint32_t* v) {
  const int* table = a.block_tables + static_cast<size_t>(it.s) * a.ld_tables;
  const int* mask = a.masks ? a.masks + static_cast<size_t>(it.r.row0 + it.first + token) * a.words : nullptr;
  for (int p = max(it.r.ctx, t0 * kKeys); p < min(it.kv_end, (t0 + take) * kKeys); ++p) {
    if (!(seen_bits(mask, a.words, it.first + token, it.r.rows, p - it.r.ctx) & 1)) continue;
    const long long at = tree::cache_row(table, p, a.num_pages);
    if (at < 0) continue;
    const bf16* value = static_cast<const bf16*>(a.kv_layer) + ((((at >> 4) * 2 + 1) * a.kv_heads + it.kvh) * 16 + (at & 15)) * kD + c1;
    for (int c = 0; c < 32; ++c) {
      const float x = __bfloat162float(value[c]);
      if (!isfinite(x)) v[c] = __float_as_uint(__uint_as_float(v[c]) + x);
    }
  }
}

// A warp's rows of an item on their way out: 32 rows of 64 bytes at a time lie in shared memory and leave it as whole sectors (a lane's own 16 bytes of 32
// rows would be 32 lines a store).
struct Rows {
  const b200_tree_attn_args* a;
  const Item* it;
  uint8_t* stage;
  int row0, rows, lane;           // the warp's first row, the item's rows
  bool whole;                     // the item's tiles were all this range's: normalised rows to the output, else fp32 ones to `part` with their maximum and sum
  int t0, take;
  bool odd;                       // infinities or NaN among its drafts' values
  float* part;

  // the output at o in TMEM; m in units of log 2
  __device__ __forceinline__ void write(uint32_t o, float m, float sum) const {
    const int group = a->q_heads / a->kv_heads, shift = __ffs(group) - 1, row = row0 + lane;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    // two rows are a line of 128 bytes, pieces of 16 bytes in an order that leaves no bank twice
    auto piece = [&](int r, int k) { return reinterpret_cast<uint4*>(stage + (r >> 1) * 128 + ((((r & 1) * 4 + k) ^ ((r >> 1) & 7)) << 4)); };
#pragma unroll
    for (int c1 = 0; c1 < kD; c1 += 32) {
      uint32_t v[32];
      tmem_ld_32x32(o + c1, v);
      tmem_ld_wait();
      if (odd && row < rows) {
        uint32_t y[32];
        for (int c = 0; c < 32; ++c) y[c] = v[c];
        add_odd(*a, *it, t0, take, c1, row >> shift, y);
        for (int c = 0; c < 32; ++c) v[c] = y[c];
      }
      auto leave = [&](int to_column, int bytes_a_value) {      // what lies there, 64 bytes a row
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2), k = lane & 3, to = row0 + r;
          const uint4 x = *piece(r, k);
          if (to >= rows) continue;
          if (bytes_a_value == 2)
            *reinterpret_cast<uint4*>(static_cast<bf16*>(a->out) + static_cast<size_t>(it->r.row0 + it->first + (to >> shift)) * a->ldo + (it->kvh * group + (to & (group - 1))) * kD + to_column + 8 * k) = x;
          else
            *reinterpret_cast<uint4*>(part + static_cast<size_t>(to) * kLd + to_column + 4 * k) = x;
        }
        __syncwarp();
      };
      if (whole) {
#pragma unroll
        for (int c = 0; c < 32; c += 8)
          *piece(lane, c / 8) =
              make_uint4(pack_bf16x2(__uint_as_float(v[c]) * inv, __uint_as_float(v[c + 1]) * inv), pack_bf16x2(__uint_as_float(v[c + 2]) * inv, __uint_as_float(v[c + 3]) * inv),
                         pack_bf16x2(__uint_as_float(v[c + 4]) * inv, __uint_as_float(v[c + 5]) * inv), pack_bf16x2(__uint_as_float(v[c + 6]) * inv, __uint_as_float(v[c + 7]) * inv));
        leave(c1, 2);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 0; c < 16; c += 4) *piece(lane, c / 4) = make_uint4(v[16 * h + c], v[16 * h + c + 1], v[16 * h + c + 2], v[16 * h + c + 3]);
          leave(c1 + 16 * h, 4);
        }
      }
    }
    if (!whole && row < rows) *reinterpret_cast<float2*>(part + static_cast<size_t>(row) * kLd + kD) = make_float2(m, sum);
  }
};

__global__ void __launch_bounds__(kThreads, kPlaces)
tree_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ b200_tree_attn_args a, float scale_log2, int* error) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t q_s = sbase, k_s = sbase + kKeysAt, v_s = sbase + kValuesAt, bars = sbase + kBars;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (2 + s); };
  auto v_full = [&](int s) { return bars + 8u * (4 + s); };
  auto v_empty = [&](int s) { return bars + 8u * (6 + s); };
  // of every other tile each: a softmax warp is up to two tiles ahead of the slowest one
  auto s_full = [&](int b) { return bars + 8u * (8 + b); };
  auto p_ready = [&](int b) { return bars + 8u * (10 + b); };
  auto pv_full = [&](int b) { return bars + 8u * (12 + b); };
  const uint32_t q_full = bars + 8u * 14, q_empty = bars + 8u * 15, slot = bars + 8u * 16;
  static_assert(kDepth == 2, "");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + (slot - sbase));
  volatile int* odd_item = reinterpret_cast<volatile int*>(tmem_slot + 2);      // [2]: the last item of each parity with infinities or NaN among its drafts' values
  __shared__ int sums[kWarps];
  __shared__ int s_range[3];        // begin, end, and the first tile of the begin's item
  __shared__ int s_where[3];
  const int warp = warp_number(), lane = threadIdx.x & 31, tid = threadIdx.x;

  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < 2; ++s) {
        mbar_init(k_full(s), 1); mbar_init(k_empty(s), 1); mbar_init(v_full(s), 1); mbar_init(v_empty(s), 1);
        mbar_init(s_full(s), 1); mbar_init(p_ready(s), 4); mbar_init(pv_full(s), 1);
      }
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      fence_mbar_init();
      odd_item[0] = odd_item[1] = -1;
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_kv);
    }
    __syncwarp();
    tmem_alloc(slot, 256);
    tmem_relinquish();
  }
  griddep_enter();
  const int ctas = gridDim.x, cta = blockIdx.x, bt = block_tokens(a);
  // ---- this CTA's range, and where it begins: every thread sums some requests, one behind the other, and the sums of the threads in front of it
  const int per_thread = (a.S + kThreads - 1) / kThreads, s_begin = min(a.S, tid * per_thread), s_end = min(a.S, s_begin + per_thread);
  int before = 0, N = 0;
  for (int s = s_begin; s < s_end; ++s) before += head_cost(a, request(a, s), bt) * a.kv_heads;
  const int own = before;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  before -= own;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int x = sums[w];
    if (w < warp) before += x;
    N += x;
  }
  const tree::Ranges ranges = tree::ranges_of(N, ctas);
  bool ok = true;
  if (N > 0 && cta < ranges.n) {
    const int b[2] = {ranges.at(cta), ranges.at(cta + 1)};
    if (tid == 0 && cta + 1 == ranges.n) s_range[1] = N;      // which lies in no item
    if (b[0] < before + own && b[1] >= before)
      for (int s = s_begin; s < s_end; ++s) {
        const tree::Request r = request(a, s);
        const int mine = head_cost(a, r, bt) * a.kv_heads;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (mine == 0 || b[e] < before || b[e] >= before + mine) continue;
          int g0 = before, block = 0, tiles = tiles_of(a, r, bt, 0);
          while (b[e] >= g0 + (tiles + tree::kItem) * a.kv_heads) g0 += (tiles + tree::kItem) * a.kv_heads, tiles = tiles_of(a, r, bt, ++block);
          const int kvh = (b[e] - g0) / (tiles + tree::kItem);
          g0 += kvh * (tiles + tree::kItem);
          s_range[e] = tree::snapped(b[e], g0, tiles, ranges.snap);
          if (e == 0) { s_where[0] = s; s_where[1] = kvh; s_where[2] = block; s_range[2] = g0; }
        }
        before += mine;
      }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tm_o = tmem + 128;
  auto tm_s = [&](int b) { return tmem + 64u * b; };
  Cut cut = {0, 0, 0, 0};
  const int left = N > 0 && cta < ranges.n ? s_range[1] - s_range[0] : 0;

  if (left > 0) {
    // every role walks the same items: item, its first tile here, and the range's cost to go
    Item it;
    it.s = s_where[0]; it.kvh = s_where[1]; it.block = s_where[2];
    it.r = request(a, it.s);
    fill(a, bt, &it);
    int t0 = max(0, s_range[0] - s_range[2] - tree::kItem), rest = left;
    auto next_item = [&] {
      if (++it.kvh >= a.kv_heads) {
        it.kvh = 0;
        if (++it.block >= blocks_of(it.r, bt)) {
          it.block = 0;
          do it.r = request(a, ++it.s);
          while (it.r.rows == 0);      // (a range's tiles are some request's: the walk ends in front of a.S)
        }
      }
      fill(a, bt, &it);
    };
    if (t0 == it.tiles) {              // the range begins where the item in front of it ends
      t0 = 0;
      next_item();
    }
    const int group = a.q_heads / a.kv_heads;
    int gt = 0, item = 0;              // tiles and items of this range so far

    if (warp == 0 || warp == kWarps - 3) {
      // ------------------------------------------------------------ loads: queries and keys, or values
      const bool one = elect_one(), values = warp != 0;
      const uint32_t ring = values ? v_s : k_s, full0 = values ? v_full(0) : k_full(0), empty0 = values ? v_empty(0) : k_empty(0);
      for (bool more = true; ok && more; ++item) {
        const uint64_t hint = it.r.rows > bt ? kEvictNormal : kEvictFirst;
        const int take = tree::take_of(t0, it.tiles, &rest), pages = (it.kv_end + 15) >> 4, p_begin = t0 * 4;
        const int* table = a.block_tables + static_cast<size_t>(it.s) * a.ld_tables;
        // the first row of a page's head; a page that the cache does not have lies behind its last row, where a load finds zeros
        auto look_up = [&](int base) {
          const int p = base + lane, page = p < pages ? table[p] : -1;
          return (((page >= 0 && page < a.num_pages ? page : static_cast<int>(a.num_pages)) * 2 + values) * a.kv_heads + it.kvh) * 16;
        };
        int mine = look_up(p_begin), next = look_up(p_begin + 32);
        if (!values) {
          if (!(ok = warp_wait(q_empty, (item & 1) ^ 1u))) break;
          if (one) {
            mbar_arrive_expect_tx(q_full, 2 * kQSlab);
            for (int h = 0; h < 2; ++h) tma_load_3d(q_s + h * kQSlab, &tm_q, q_full, 64 * h, it.kvh * group, it.r.row0 + it.first);
          }
        }
        for (int j = 0; j < take; ++j, ++gt) {
          if (j && j % 8 == 0) {
            mine = next;
            next = look_up(p_begin + 4 * j + 32);
          }
          const int n = min(4, pages - p_begin - 4 * j), st = gt & 1;
          int row[4];
#pragma unroll
          for (int pg = 0; pg < 4; ++pg) row[pg] = __shfl_sync(0xffffffffu, mine, (4 * j + pg) & 31);
          if (!(ok = warp_wait(empty0 + 8 * st, ((gt >> 1) & 1) ^ 1u))) break;
          const uint32_t full = full0 + 8 * st, dst = ring + st * kTile;
          if (one) {
            mbar_arrive_expect_tx(full, n * 4096);
#pragma unroll
            for (int pg = 0; pg < 4; ++pg) {
              if (pg >= n) break;
              tma_load_2d(dst + pg * 2048, &tm_kv, full, 0, row[pg], hint);
              tma_load_2d(dst + kSlab + pg * 2048, &tm_kv, full, 64, row[pg], hint);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        if (rest == 0 && t0 == 0 && take < it.tiles) cut = {it.r.row0 + it.first, it.nb * group, it.kvh, ranges.parts(cta, s_range[1] - take, it.tiles)};
        t0 = 0;
        if ((more = rest > 0)) next_item();
      }
      // the copies in flight land before the CTA ends, also where it gives up
      if (!values && item + !ok > 0) warp_wait(q_full, (item - ok) & 1);
      for (int k = max(0, gt - kDepth); k < gt; ++k) warp_wait(full0 + 8 * (k & 1), (k >> 1) & 1);
    } else if (warp == kWarps - 2) {
      // ------------------------------------------------------------ scores
      const bool one = elect_one();
      const uint32_t id_s = idesc_bf16(kRows, kKeys, 0);
      const uint64_t q_d = desc_sw128(q_s, 16, 1024), k_d = desc_sw128(k_s, 16, 1024);
      for (bool more = true; ok && more; ++item) {
        const int take = tree::take_of(t0, it.tiles, &rest);
        if (!(ok = warp_wait(q_full, item & 1))) break;
        for (int j = 0; j < take; ++j, ++gt) {
          const int b = gt & 1;
          // the keys are there, and the buffer's last P has been read by the products with its values
          if (!(ok = warp_wait(k_full(b), (gt >> 1) & 1) && (gt < 2 || warp_wait(pv_full(b), ((gt - 2) >> 1) & 1)))) break;
          tc_fence_after();
          if (one) {
#pragma unroll
            for (int h = 0; h < 2; ++h) umma_bf16_k64(tm_s(b), q_d + h * (kQSlab >> 4), k_d + b * (kTile >> 4) + h * (kSlab >> 4), id_s, h);
            umma_commit(s_full(b));
            umma_commit(k_empty(b));
            if (j + 1 == take) umma_commit(q_empty);
          }
          __syncwarp();
        }
        if (!ok) break;
        t0 = 0;
        if ((more = rest > 0)) next_item();
      }
      if (!ok && gt) warp_wait(s_full((gt - 1) & 1), ((gt - 1) >> 1) & 1);      // no product is under way when tensor memory is given back
    } else if (warp == kWarps - 1) {
      // ------------------------------------------------------------ outputs
      const bool one = elect_one();
      const uint32_t id_o = idesc_bf16(kRows, kD, 1);
      const uint64_t v_d = desc_sw128(v_s, kSlab, 1024);
      for (bool more = true; ok && more; ++item) {
        const int take = tree::take_of(t0, it.tiles, &rest);
        for (int j = 0; j < take; ++j, ++gt) {
          const int b = gt & 1, kv0 = (t0 + j) * kKeys;
          if (!(ok = warp_wait(v_full(b), (gt >> 1) & 1))) break;
          if (kv0 + kKeys > it.r.ctx) {
            bool odd = false;
            const int from = max(0, it.r.ctx - kv0), end = min(kKeys, it.kv_end - kv0);      // the drafts' rows of the tile
            for (int h = 0; h < 2; ++h) {
              uint4* v = reinterpret_cast<uint4*>(smem + (v_s - sbase) + b * kTile + h * kSlab);      // (a row's pieces in some order)
              for (int e0 = from * 8; e0 < end * 8; e0 += 256) {
                uint4 x[8];
                uint32_t any = 0;      // bit 15 or 31: an exponent of all ones
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = v[min(e0 + 32 * k + lane, end * 8 - 1)];
                auto carry = [](uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; };
#pragma unroll
                for (int k = 0; k < 8; ++k) any |= carry(x[k].x) | carry(x[k].y) | carry(x[k].z) | carry(x[k].w);
                if (any & 0x80008000u) {
                  odd = true;
#pragma unroll
                  for (int k = 0; k < 8; ++k) v[min(e0 + 32 * k + lane, end * 8 - 1)] = make_uint4(without_odd(x[k].x), without_odd(x[k].y), without_odd(x[k].z), without_odd(x[k].w));
                }
              }
              for (int e = end * 8 + lane; e < kKeys * 8; e += 32) v[e] = make_uint4(0, 0, 0, 0);
            }
            if (odd) odd_item[item & 1] = item;
            __threadfence_block();
            fence_proxy_async();
            __syncwarp();
          }
          if (!(ok = warp_wait(p_ready(b), (gt >> 1) & 1))) break;
          tc_fence_after();
          if (one) {
            umma_bf16_tmem_k64(tm_o, tm_s(b), v_d + b * (kTile >> 4), id_o, j > 0);
            umma_commit(pv_full(b));
            umma_commit(v_empty(b));
          }
          __syncwarp();
        }
        if (!ok) break;
        t0 = 0;
        if ((more = rest > 0)) next_item();
      }
      if (!ok && gt) warp_wait(pv_full((gt - 1) & 1), ((gt - 1) >> 1) & 1);
    } else {
      // ------------------------------------------------------------ softmax: thread = row (token * group + head)
      const int q = warp & 3, row = q * 32 + lane;      // the quarter of the lanes that this warp may access
      const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
      for (bool more = true; ok && more; ++item) {
        const int take = tree::take_of(t0, it.tiles, &rest), rows = it.nb * group;
        const bool valid = row < rows, some = row - lane < rows;      // this warp has rows
        const int token = it.first + row / group;
        const int* mask = a.masks && valid ? a.masks + static_cast<size_t>(it.r.row0 + token) * a.words : nullptr;
        float ref = -INFINITY, l = 0.f;      // what the row's weights are relative to, in units of log 2, and their sum
        for (int j = 0; j < take; ++j, ++gt) {
          const int b = gt & 1, kv0 = (t0 + j) * kKeys;
          if (!(ok = warp_wait(s_full(b), (gt >> 1) & 1))) break;
          if (some) {
            tc_fence_after();
            uint32_t s0[32], s1[32];
            tmem_ld_32x32(tm_s(b) + lane_off, s0);
            tmem_ld_32x32(tm_s(b) + lane_off + 32, s1);
            tmem_ld_wait();
            if (kv0 + kKeys > it.r.ctx) {
              const uint32_t m0 = valid ? seen_bits(mask, a.words, token, it.r.rows, kv0 - it.r.ctx) : 0u, m1 = valid ? seen_bits(mask, a.words, token, it.r.rows, kv0 + 32 - it.r.ctx) : 0u;
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                if (!(m0 >> c & 1)) s0[c] = 0xff800000u;
                if (!(m1 >> c & 1)) s1[c] = 0xff800000u;
              }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 32; c += 2)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                mx[k] = fmaxf(mx[k], __uint_as_float(s0[c + k]));
                mx[2 + k] = fmaxf(mx[2 + k], __uint_as_float(s1[c + k]));
              }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2;
            float alpha = 1.f;
            if (top > ref) {
              alpha = exp2_ftz(ref - top);
              ref = top;
            }
            const float mu = ref == -INFINITY ? 0.f : ref;
            auto weight = [&](uint32_t w) { return exp2_ftz(fmaf(__uint_as_float(w), scale_log2, -mu)); };
            float ps = 0.f;
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const uint32_t a0 = pack_bf16x2(weight(s0[c]), weight(s0[c + 1])), a1 = pack_bf16x2(weight(s1[c]), weight(s1[c + 1]));
              // the sum is that of the rounded weights: where one weight outweighs the others, its rounding cancels
              ps += (__uint_as_float(a0 << 16) + __uint_as_float(a0 & 0xffff0000u)) + (__uint_as_float(a1 << 16) + __uint_as_float(a1 & 0xffff0000u));
              pk[c >> 1] = a0;
              pk[16 + (c >> 1)] = a1;
            }
            l = l * alpha + ps;
            // P in place of the scores: what read this buffer's last P went ahead of them.  Where some row of the warp moved its maximum, its output so
            // far is scaled once the previous product has landed.
            tmem_st_32x32(tm_s(b) + lane_off, pk);
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
              if (!(ok = warp_wait(pv_full(b ^ 1), ((gt - 1) >> 1) & 1))) break;
              tc_fence_after();
#pragma unroll
              for (int c0 = 0; c0 < kD; c0 += 32) {
                uint32_t v[32];
                tmem_ld_32x32(tm_o + lane_off + c0, v);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * alpha);
                tmem_st_32x32(tm_o + lane_off + c0, v);
              }
            }
            tmem_st_wait();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(p_ready(b));
        }
        if (!ok) break;
        // ---- the item's rows
        if (!(ok = warp_wait(pv_full((gt - 1) & 1), ((gt - 1) >> 1) & 1))) break;
        tc_fence_after();
        if (some) {
          Rows out{&a, &it, smem + kStageAt + q * 2048, q * 32, rows, lane, t0 == 0 && take == it.tiles, t0, take, odd_item[item & 1] == item, nullptr};
          out.part = rows_of(a.workspace, ctas) + static_cast<size_t>(2 * cta + (t0 == 0)) * kRows * kLd;      // a part without the item's beginning is the range's first
          out.write(tm_o + lane_off, ref, l);
        }
        tc_fence_before();
        t0 = 0;
        if ((more = rest > 0)) next_item();
      }
    }
  }
  if (tid == 0) reinterpret_cast<Cut*>(a.workspace)[cta] = cut;
  if (!ok) *reinterpret_cast<volatile int*>(error) = 1;
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// A row of an item that ranges' ends cut: sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p over the parts, in order, four dimensions a lane: the form for few parts.
template <typename Part>
__device__ __forceinline__ void join_few(int parts, Part part, int lane, uint2* out) {
  float m = -INFINITY, sum = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += kFew) {
    float2 st[kFew];
    float4 x[kFew];
    float top = m;
#pragma unroll
    for (int k = 0; k < kFew; ++k) {
      const bool there = p0 + k < parts;
      st[k] = there ? *reinterpret_cast<const float2*>(part(p0 + k) + kD) : make_float2(-INFINITY, 0.f);
      x[k] = there ? *reinterpret_cast<const float4*>(part(p0 + k) + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < kFew; ++k) top = fmaxf(top, st[k].x);
    const float base = top == -INFINITY ? 0.f : top, old = exp2f(m - base);
    m = top;
    sum *= old;
    y = make_float4(y.x * old, y.y * old, y.z * old, y.w * old);
#pragma unroll
    for (int k = 0; k < kFew; ++k) {
      const float w = exp2f(st[k].x - base);
      sum += w == 0.f && st[k].y == st[k].y ? 0.f : st[k].y * w;
      if (w != 0.f) y = make_float4(fmaf(x[k].x, w, y.x), fmaf(x[k].y, w, y.y), fmaf(x[k].z, w, y.z), fmaf(x[k].w, w, y.w));
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *out = make_uint2(pack_bf16x2(y.x * inv, y.y * inv), pack_bf16x2(y.z * inv, y.w * inv));
}

// The form for many: a lane has the maximum, sum and weight of one part in 32.
template <typename Part>
__device__ __forceinline__ void join_row(int parts, Part part, int lane, uint2* out) {
  float m = -INFINITY, sum = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += 32) {
    const int n = min(32, parts - p0);
    const float2 st = lane < n ? *reinterpret_cast<const float2*>(part(p0 + lane) + kD) : make_float2(-INFINITY, 0.f);
    float4 x[kJoinAtOnce];
    auto load = [&](int k0) {
#pragma unroll
      for (int k = 0; k < kJoinAtOnce; ++k)
        if (k0 + k < n) x[k] = *reinterpret_cast<const float4*>(part(p0 + k0 + k) + lane * 4);
    };
    load(0);
    float top = fmaxf(m, st.x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top, old = exp2f(m - base), w = exp2f(st.x - base);
    m = top;
    float l = w == 0.f && st.y == st.y ? 0.f : st.y * w;
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    sum = sum * old + l;
    y = make_float4(y.x * old, y.y * old, y.z * old, y.w * old);
    for (int k0 = 0; k0 < n; k0 += kJoinAtOnce) {
      if (k0) load(k0);
#pragma unroll
      for (int k = 0; k < kJoinAtOnce; ++k) {
        const float wk = __shfl_sync(0xffffffffu, w, (k0 + k) & 31);
        if (k0 + k < n && wk != 0.f) y = make_float4(fmaf(x[k].x, wk, y.x), fmaf(x[k].y, wk, y.y), fmaf(x[k].z, wk, y.z), fmaf(x[k].w, wk, y.w));
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *out = make_uint2(pack_bf16x2(y.x * inv, y.y * inv), pack_bf16x2(y.z * inv, y.w * inv));
}

// All such rows, a warp each: every block sums the cut items' rows for itself and takes its share.  What bounds it is the chain from the first kernel's end (the cuts,
// a search, statistics, parts): 3 us of a call of 1 x 450, 6 of 64 x 2048, 5 of 2 x 32001, 11 of 48 x 1999 with 64 rows, whose parts are 19 MB.  A block for eight rows of each CTA's item,
// of which most had none, came in eleven waves and with the form of twelve parts at once for every row: 2, 4.5 and 8 us more.
__global__ void __launch_bounds__(kJoinThreads, kJoinPlaces)
tree_attn_join_kernel(const __grid_constant__ b200_tree_attn_args a, int ctas, int blocks) {
  extern __shared__ int rows_before[];      // [ctas + 1] of each CTA's cut item
  __shared__ int sums[kJoinThreads / 32];
  griddep_enter();
  if (static_cast<int>(blockIdx.x) >= blocks) return zero_rest(a, blockIdx.x - blocks, gridDim.x - blocks);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = a.q_heads / a.kv_heads;
  const Cut* cuts = static_cast<const Cut*>(a.workspace);
  const int per = (ctas + kJoinThreads - 1) / kJoinThreads, begin = min(ctas, tid * per), end = min(ctas, begin + per);
  int before = 0, all = 0;
  for (int c = begin; c < end; ++c) before += cuts[c].parts ? cuts[c].rows : 0;
  const int own = before;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  before -= own;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  for (int c = begin; c < end; ++c) {
    rows_before[c] = before;
    before += cuts[c].parts ? cuts[c].rows : 0;
  }
  if (tid == 0) rows_before[ctas] = all;
  __syncthreads();
  const float* ws = rows_of(a.workspace, ctas);
  for (int n = blockIdx.x * (kJoinThreads / 32) + warp; n < all; n += blocks * (kJoinThreads / 32)) {
    const int c = tree::last_at_most(rows_before, ctas, n), row = n - rows_before[c];
    const Cut cut = cuts[c];
    // the item's beginning lies in its range's second place, each other part in its range's first
    auto part = [&](int p) { return ws + (static_cast<size_t>(2 * (c + p) + (p == 0)) * kRows + row) * kLd; };
    uint2* out = reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + static_cast<size_t>(cut.row0 + row / group) * a.ldo + (cut.kvh * group + row % group) * kD + lane * 4);
    if (cut.parts <= kFew) join_few(cut.parts, part, lane, out);
    else join_row(cut.parts, part, lane, out);
  }
}

}  // namespace

int64_t tree_attention_workspace(const b200_tree_attn_args&) { return static_cast<int64_t>(kPlaces) * sm_count() * (static_cast<int64_t>(sizeof(Cut)) + 2ll * kRows * kLd * sizeof(float)); }

int paged_attention_tree(const b200_tree_attn_args& a, int* error, cudaStream_t st) {
  const int group = a.q_heads / a.kv_heads;
  const int rows = static_cast<int>(std::min(static_cast<long long>(kRows), std::min(a.max_tree, a.T) * static_cast<long long>(group)));
  // as many CTAs as there are places, or as the most work that the call may have feeds: 0.6 us less for 1 x 450 (11.0 now) than over all places
  const long long seen = std::min(a.max_ctx ? a.max_ctx : INT_MAX, a.max_blocks * tree::kPage) + static_cast<long long>(std::min(a.max_tree, a.T));
  const long long items = (static_cast<long long>(std::min(a.max_tree, a.T)) * group + kRows - 1) / kRows * a.kv_heads * a.S, cost = items * ((seen + kKeys - 1) / kKeys + tree::kItem);
  const int ctas = static_cast<int>(std::min<long long>(kPlaces * sm_count(), std::max<long long>(1, cost / tree::kLeast)));
  CUtensorMap tm_q, tm_kv;
  if (int rc = tmap_encode_bf16_3d(&tm_q, a.q, kD, a.q_heads, a.T, kD, a.ldq, 64, group, kRows / group)) return rc;
  if (int rc = tmap_encode_bf16_2d(&tm_kv, a.kv_layer, static_cast<uint64_t>(a.num_pages) * 2 * a.kv_heads * 16, kD, kD, 16, 64, 1)) return rc;
  static std::atomic<unsigned long long> attr_done{0};
  if (!ensure_dynamic_smem(tree_attn_kernel, kSmem, &attr_done)) return -3;
  launch_pdl(tree_attn_kernel, dim3(ctas), dim3(kThreads), kSmem, st, tm_q, tm_kv, a, a.scale * 1.4426950408889634f, error);
  if (cudaGetLastError() != cudaSuccess) return -2;
  const int blocks = std::min(kJoinPlaces * sm_count(), (ctas * rows + kJoinThreads / 32 - 1) / (kJoinThreads / 32));
  const int zeros = a.zero_rest ? std::min(64, a.T / 16 + 1) : 0;      // blocks behind those
  launch_pdl(tree_attn_join_kernel, dim3(blocks + zeros), dim3(kJoinThreads), (ctas + 1) * sizeof(int), st, a, ctas, blocks);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
