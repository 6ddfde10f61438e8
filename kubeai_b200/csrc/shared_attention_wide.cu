// Attention of parts of many rows, on the 5th-generation tensor cores: a group's rows over the pages that it shares, and the own keys of requests with long chains
// (shared_attention.cu has the parts, the joining and what parts of few rows take).
//
// An item is a part's key head and up to 128 of its rows (row = token * group + head); its keys come in tiles of 64.  All items' tiles one behind the other are cut into as many equal ranges as
// the SMs have places for CTAs, two each, and a CTA walks its range without a gap:
//   two warps look pages up (32 of the table at a time, the next ones ahead) and load by TMA, 128-byte swizzle, into rings, one queries and keys, one values;
//   two warps issue tcgen05.mma, one S = Q K^T (M = 128, N = 64, two buffers), one O += P V (M = 128, N = 128, P in TMEM over its scores);
//   four warps (thread = row) do the softmax in fp32, base 2; a warp whose rows nobody owns only keeps step.
// Weights are relative to the row's largest score so far, so the largest weight is exactly 1 and its rounding to bf16 costs nothing.
// Only tiles that reach behind what every row sees are masked.  There the products' warp also clears what must not meet a weight of zero: values behind the last key, and infinities and NaN
// among values that some row does not see, which the rows that see them add at the end by themselves.
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
#include "shared_attention.cuh"

namespace b200 {
namespace {

typedef __nv_bfloat16 bf16;
using namespace shared_attn;
typedef Items<true> I;
constexpr int kRows = kWideRows, kKeys = I::kUnit;
constexpr int kQSlab = kRows * 128, kSlab = kKeys * 128, kTile = 2 * kSlab;      // bytes: 64 columns of a row tile, of a key tile, a key tile
constexpr int kThreads = 256, kWarps = kThreads / 32, kPlaces = 2;                // kPlaces: CTAs of an SM
constexpr int kDepth = 2;                  // tiles of keys, and of values, on their way

// shared memory: queries, keys, values, 2 KB a softmax warp for its way out, barriers
constexpr int kKeysAt = 2 * kQSlab, kValuesAt = kKeysAt + kDepth * kTile, kStageAt = kValuesAt + kDepth * kTile, kBars = kStageAt + 4 * 2048, kSmem = 1024 + kBars + 256;
static_assert(kPlaces * (kSmem + 1024 + 128) <= 228 * 1024, "");

// An item of a range as all roles see it
struct View {
  int end, see;      // keys behind the last, and behind the last that the block's token 0 sees; token i sees i more
  int rows, row0;    // token * group + head; the block's first row of the step
  __device__ __forceinline__ View(const Item<true>& it, int group)
      : end(it.k1), see(it.p.all ? it.k1 : it.p.ctx + it.first + 1), rows(it.nb * group), row0(it.p.row0 + it.first) {}
  __device__ __forceinline__ int limit(int token) const { return min(see + token, end); }
};

// Infinities and NaN among values that a row sees and others do not, which stayed out of the products, to its dimensions c1 ..
__device__ __noinline__ void add_odd(const b200_shared_attn_args& a, int table_row, int kvh, int from, int limit, int c1, uint32_t* v) {
  const int* table = a.block_tables + static_cast<size_t>(table_row) * a.ld_tables;
  for (int p = from; p < limit; ++p) {
    const long long at = tree::cache_row(table, p, a.num_pages);
    if (at < 0) continue;
    const bf16* value = static_cast<const bf16*>(a.kv_layer) + ((((at >> 4) * 2 + 1) * a.kv_heads + kvh) * 16 + (at & 15)) * kD + c1;
    for (int c = 0; c < 32; ++c) {
      const float x = __bfloat162float(value[c]);
      if (!isfinite(x)) v[c] = __float_as_uint(__uint_as_float(v[c]) + x);
    }
  }
}

// A warp's rows of an item on their way out: 32 rows of 64 bytes at a time lie in shared memory and leave it as whole sectors (a lane's own 16 bytes of 32
// rows would be 32 lines a store).
struct Rows {
  const b200_shared_attn_args* a;
  const Item<true>* it;
  uint8_t* stage;
  int row0, rows, lane;           // the warp's first row, the item's rows
  int group, shift;
  float* part;                    // fp32 rows with their maximum and sum: the range's slot, or null for the rows of all
  float* all;
  bool last;                      // normalised rows to the output
  int odd_from, odd_to;           // keys whose odd values this thread's row adds

  __device__ __forceinline__ float* row_at(int to) const {
    if (part) return part + static_cast<size_t>(to) * kLd;
    return all + ((static_cast<size_t>(!it->p.all) * a->T + it->p.row0 + it->first + (to >> shift)) * a->q_heads + it->kvh * group + (to & (group - 1))) * kLd;
  }
  // the output at o in TMEM; m in units of log 2
  __device__ __forceinline__ void write(uint32_t o, float m, float sum) const {
    const int row = row0 + lane;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    // two rows are a line of 128 bytes, pieces of 16 bytes in an order that leaves no bank twice
    auto piece = [&](int r, int k) { return reinterpret_cast<uint4*>(stage + (r >> 1) * 128 + ((((r & 1) * 4 + k) ^ ((r >> 1) & 7)) << 4)); };
#pragma unroll
    for (int c1 = 0; c1 < kD; c1 += 32) {
      uint32_t v[32];
      tmem_ld_32x32(o + c1, v);
      tmem_ld_wait();
      if (odd_from < odd_to && row < rows) {
        uint32_t y[32];
        for (int c = 0; c < 32; ++c) y[c] = v[c];
        add_odd(*a, it->p.table, it->kvh, odd_from, odd_to, c1, y);
        for (int c = 0; c < 32; ++c) v[c] = y[c];
      }
      auto leave = [&](int to_column) {      // what lies there, 64 bytes a row
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2), k = lane & 3, to = row0 + r;
          const uint4 x = *piece(r, k);
          if (to >= rows) continue;
          if (last)
            *reinterpret_cast<uint4*>(static_cast<bf16*>(a->out) + static_cast<size_t>(it->p.row0 + it->first + (to >> shift)) * a->ldo + (it->kvh * group + (to & (group - 1))) * kD + to_column + 8 * k) = x;
          else
            *reinterpret_cast<uint4*>(row_at(to) + to_column + 4 * k) = x;
        }
        __syncwarp();
      };
      if (last) {
#pragma unroll
        for (int c = 0; c < 32; c += 8)
          *piece(lane, c / 8) =
              make_uint4(pack_bf16x2(__uint_as_float(v[c]) * inv, __uint_as_float(v[c + 1]) * inv), pack_bf16x2(__uint_as_float(v[c + 2]) * inv, __uint_as_float(v[c + 3]) * inv),
                         pack_bf16x2(__uint_as_float(v[c + 4]) * inv, __uint_as_float(v[c + 5]) * inv), pack_bf16x2(__uint_as_float(v[c + 6]) * inv, __uint_as_float(v[c + 7]) * inv));
        leave(c1);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 0; c < 16; c += 4) *piece(lane, c / 4) = make_uint4(v[16 * h + c], v[16 * h + c + 1], v[16 * h + c + 2], v[16 * h + c + 3]);
          leave(c1 + 16 * h);
        }
      }
    }
    if (!last && row < rows) *reinterpret_cast<float2*>(row_at(row) + kD) = make_float2(m, sum);
  }
};

__global__ void __launch_bounds__(kThreads, kPlaces)
shared_attn_wide_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ b200_shared_attn_args a, const Sizes sizes, float scale_log2,
                        int* error) {
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
  volatile int* odd_item = reinterpret_cast<volatile int*>(tmem_slot + 2);      // [2]: the last item of each parity with infinities or NaN among values that some row does not see
  __shared__ int sums[kWarps], s_range[2], s_where[2][4];
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
  const int cta = blockIdx.x, group = a.q_heads / a.kv_heads, shift = __ffs(group) - 1, bt = kRows / group;
  bool ordered = a.G > 0;
  if (ordered) ordered = __syncthreads_and(beam::ascends(a.group_starts, a.G, a.S, tid, kThreads) && beam::ascends(a.starts, a.S, a.T, tid, kThreads));
  const Lengths n = lengths_of(a, ordered);
  const tree::Ranges ranges = find_ranges<true, kThreads>(n, a.kv_heads, group, cta, 1, sizes.ctas, sums, s_range, s_where);
  bool ok = true;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tm_o = tmem + 128;
  auto tm_s = [&](int b) { return tmem + 64u * b; };
  const int left = cta < ranges.n ? s_range[1] - s_range[0] : 0;

  if (left > 0) {
    // every role walks the same items: item, its first tile here, and the range's cost to go
    Item<true> it;
    it.u = s_where[0][0]; it.kvh = s_where[0][1]; it.block = s_where[0][2];
    it.p = I::part(n, it.u, group);
    it.fill(bt);
    int t0 = max(0, s_range[0] - s_where[0][3] - tree::kItem), rest = left;
    if (t0 == it.units) {              // the range begins where the item in front of it ends
      t0 = 0;
      it.next(n, a.kv_heads, group, bt);
    }
    int gt = 0, item = 0;              // tiles and items of this range so far

    if (warp == 0 || warp == kWarps - 3) {
      // ------------------------------------------------------------ loads: queries and keys, or values
      const bool one = elect_one(), values = warp != 0;
      const uint32_t ring = values ? v_s : k_s, full0 = values ? v_full(0) : k_full(0), empty0 = values ? v_empty(0) : k_empty(0);
      for (bool more = true; ok && more; ++item) {
        const uint64_t hint = it.p.rows > bt ? kEvictNormal : kEvictFirst;
        const int take = tree::take_of(t0, it.units, &rest), pages = (it.k1 - it.p.k0 + 15) >> 4, p_begin = t0 * 4;
        const int* table = a.block_tables + static_cast<size_t>(it.p.table) * a.ld_tables + it.p.k0 / 16;
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
            for (int h = 0; h < 2; ++h) tma_load_3d(q_s + h * kQSlab, &tm_q, q_full, 64 * h, it.kvh * group, it.p.row0 + it.first);
          }
        }
        for (int j = 0; j < take; ++j, ++gt) {
          if (j && j % 8 == 0) {
            mine = next;
            next = look_up(p_begin + 4 * j + 32);
          }
          const int count = min(4, pages - p_begin - 4 * j), st = gt & 1;
          int row[4];
#pragma unroll
          for (int pg = 0; pg < 4; ++pg) row[pg] = __shfl_sync(0xffffffffu, mine, (4 * j + pg) & 31);
          if (!(ok = warp_wait(empty0 + 8 * st, ((gt >> 1) & 1) ^ 1u))) break;
          const uint32_t full = full0 + 8 * st, dst = ring + st * kTile;
          if (one) {
            mbar_arrive_expect_tx(full, count * 4096);
#pragma unroll
            for (int pg = 0; pg < 4; ++pg) {
              if (pg >= count) break;
              tma_load_2d(dst + pg * 2048, &tm_kv, full, 0, row[pg], hint);
              tma_load_2d(dst + kSlab + pg * 2048, &tm_kv, full, 64, row[pg], hint);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        if (!values && t0 == 0) {      // where the item's rows are: their tokens', 32 at a time
          const bool whole = take == it.units;
          const Place x = {2 * cta + 1, whole ? 0 : ranges.parts(cta, s_range[1] - take, it.units), 0, kWide | (it.p.k0 > 0 ? kJoined : 0)};
          for (int i = lane; i < it.nb; i += 32) {
            Place y = x;
            y.row = i << shift;
            space_of(a, sizes).places[(static_cast<size_t>(!it.p.all) * a.T + it.p.row0 + it.first + i) * a.kv_heads + it.kvh] = y;
          }
        }
        t0 = 0;
        if ((more = rest > 0)) it.next(n, a.kv_heads, group, bt);
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
        const int take = tree::take_of(t0, it.units, &rest);
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
        if ((more = rest > 0)) it.next(n, a.kv_heads, group, bt);
      }
      if (!ok && gt) warp_wait(s_full((gt - 1) & 1), ((gt - 1) >> 1) & 1);      // no product is under way when tensor memory is given back
    } else if (warp == kWarps - 1) {
      // ------------------------------------------------------------ outputs
      const bool one = elect_one();
      const uint32_t id_o = idesc_bf16(kRows, kD, 1);
      const uint64_t v_d = desc_sw128(v_s, kSlab, 1024);
      for (bool more = true; ok && more; ++item) {
        const int take = tree::take_of(t0, it.units, &rest);
        const View x(it, group);
        for (int j = 0; j < take; ++j, ++gt) {
          const int b = gt & 1, kv0 = it.p.k0 + (t0 + j) * kKeys;
          if (!(ok = warp_wait(v_full(b), (gt >> 1) & 1))) break;
          if (kv0 + kKeys > x.see) {
            bool odd = false;
            const int from = max(0, x.see - kv0), end = min(kKeys, x.end - kv0);      // the tile's values that some row does not see
            for (int h = 0; h < 2; ++h) {
              uint4* v = reinterpret_cast<uint4*>(smem + (v_s - sbase) + b * kTile + h * kSlab);      // (a row's pieces in some order)
              for (int e = from * 8 + lane; e < end * 8; e += 32) {
                const uint4 was = v[e], w = make_uint4(without_odd(was.x), without_odd(was.y), without_odd(was.z), without_odd(was.w));
                if (w.x != was.x || w.y != was.y || w.z != was.z || w.w != was.w) {
                  odd = true;
                  v[e] = w;
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
        if ((more = rest > 0)) it.next(n, a.kv_heads, group, bt);
      }
      if (!ok && gt) warp_wait(pv_full((gt - 1) & 1), ((gt - 1) >> 1) & 1);
    } else {
      // ------------------------------------------------------------ softmax: thread = row (token * group + head)
      const int q = warp & 3, row = q * 32 + lane;      // the quarter of the lanes that this warp may access
      const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
      for (bool more = true; ok && more; ++item) {
        const int take = tree::take_of(t0, it.units, &rest);
        const View x(it, group);
        const bool valid = row < x.rows, some = row - lane < x.rows;      // this warp has rows
        const int limit = valid ? x.limit(row >> shift) : 0;
        float ref = -INFINITY, l = 0.f;      // what the row's weights are relative to, in units of log 2, and their sum
        for (int j = 0; j < take; ++j, ++gt) {
          const int b = gt & 1, kv0 = it.p.k0 + (t0 + j) * kKeys;
          if (!(ok = warp_wait(s_full(b), (gt >> 1) & 1))) break;
          if (some) {
            tc_fence_after();
            uint32_t s0[32], s1[32];
            tmem_ld_32x32(tm_s(b) + lane_off, s0);
            tmem_ld_32x32(tm_s(b) + lane_off + 32, s1);
            tmem_ld_wait();
            if (kv0 + kKeys > x.see) {
              const int seen = limit - kv0;
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                if (c >= seen) s0[c] = 0xff800000u;
                if (c + 32 >= seen) s1[c] = 0xff800000u;
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
          const Space space = space_of(a, sizes);
          const bool whole = t0 == 0 && take == it.units, odd = odd_item[item & 1] == item;
          const int begin = it.p.k0 + t0 * kKeys;
          // a part without the item's beginning is the range's first
          Rows out{&a, &it, smem + kStageAt + q * 2048, q * 32, x.rows, lane, group, shift, whole ? nullptr : space.wide + static_cast<size_t>(2 * cta + (t0 == 0)) * kRows * kLd, space.rows,
                   whole && !it.p.all && it.p.k0 == 0, odd ? max(x.see, begin) : 0, odd ? min(limit, begin + take * kKeys) : 0};
          out.write(tm_o + lane_off, ref, l);
        }
        tc_fence_before();
        t0 = 0;
        if ((more = rest > 0)) it.next(n, a.kv_heads, group, bt);
      }
    }
  }
  if (!ok) *reinterpret_cast<volatile int*>(error) = 1;
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

}  // namespace

int shared_attention_wide_ctas(const b200_shared_attn_args& a) {
  const long long group = a.q_heads / a.kv_heads, T = a.T, most = std::min<long long>(a.max_rows, T);
  const bool shared = a.G && T * group > kNarrow, own = most * group > kNarrow;
  if (!shared && !own) return 0;
  // as many CTAs as there are places, or as the most work that the call may have feeds
  const long long seen = std::min<long long>(a.max_ctx ? a.max_ctx : INT_MAX, a.max_blocks * static_cast<long long>(tree::kPage)) + most;
  const long long items = ((shared ? (T * group + kRows - 1) / kRows + a.G : 0) + (own ? (most * group + kRows - 1) / kRows * a.S : 0)) * a.kv_heads, cost = items * ((seen + kKeys - 1) / kKeys + tree::kItem);
  return static_cast<int>(std::min<long long>(kPlaces * sm_count(), std::max<long long>(1, cost / tree::kLeast)));
}

int shared_attention_wide(const b200_shared_attn_args& a, const Sizes& sizes, int* error, cudaStream_t st) {
  const int group = a.q_heads / a.kv_heads;
  CUtensorMap tm_q, tm_kv;
  if (int rc = tmap_encode_bf16_3d(&tm_q, a.q, kD, a.q_heads, a.T, kD, a.ldq, 64, group, kRows / group)) return rc;
  if (int rc = tmap_encode_bf16_2d(&tm_kv, a.kv_layer, static_cast<uint64_t>(a.num_pages) * 2 * a.kv_heads * 16, kD, kD, 16, 64, 1)) return rc;
  static std::atomic<unsigned long long> attr_done{0};
  if (!ensure_dynamic_smem(shared_attn_wide_kernel, kSmem, &attr_done)) return -3;
  launch_pdl(shared_attn_wide_kernel, dim3(sizes.ctas), dim3(kThreads), kSmem, st, tm_q, tm_kv, a, sizes, a.scale * 1.4426950408889634f, error);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
