// Attention of the rows of drafted trees over the paged cache, on the 5th-generation tensor cores.
//
//   out_t = sum_j softmax_j(scale q_t . k_j) v_j   over j < ctx and those j = ctx + i whose bit i the row's mask has
//
// A request's rows share all keys but the last few, so what counts is that K and V pass once for all of a key head's rows: a CTA takes up to 128 * NT
// of them (row = token * group + head), its share of the context in tiles of 64 keys, and works as the kernels of chunks and prompts do:
//   one warp looks pages up (32 of the table at a time) and loads tiles by TMA, 128-byte swizzle, keys and values in rings of their own;
//   one warp issues every tcgen05.mma:  S_i = Q_i K^T (M = 128, N = 64, two buffers in TMEM),  O_i += P_i V (M = 128, N = 128, P_i in TMEM over its scores);
//   four warps a row tile (thread = row) do the softmax in fp32, base 2; warps whose rows nobody owns sleep.
// The masks' bits are looked at only in tiles that reach behind the context.  There the products' warp also clears what must not meet a weight of zero:
// values behind the last key, and infinities and NaN among the drafts' values, which the rows that see them add at the end by themselves.
// Few requests: a cluster of CTAs shares a context, each leaves its unnormalised rows in its shared memory, and the rows are joined through
// distributed shared memory in a fixed order; no workspace, one launch, the same bits every time.
// Every wait has a limit; a CTA that gives up sets an error mark and still meets at the barriers.
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
#include "umma2.cuh"

namespace b200 {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int kD = 128, kRows = 128, kKeys = 64;
constexpr int kQSlab = kRows * 128, kSlab = kKeys * 128, kTile = 2 * kSlab;      // bytes: 64 columns of a row tile, of a key tile, a key tile
constexpr int kLd = kD + 4;                                                      // floats from row to row of what a cluster joins: no bank twice
constexpr int kWaitLimit = 1 << 22;
constexpr int kMostParts = 8;

template <int NT>
struct Shape {
  static constexpr int kStages = NT == 1 ? 2 : 4;               // of keys and of values
  static constexpr int kThreads = 32 * (4 * NT + 2);
  static constexpr int kCtas = NT == 1 ? 2 : 1;                 // an SM
  static constexpr int kRing = NT * 2 * kQSlab;                 // where the keys begin
  static constexpr int kBars = kRing + 2 * kStages * kTile;
  static constexpr int kSmem = 1024 + kBars + 512;
  static_assert(NT * kRows * (kLd + 2) * 4 <= kBars, "rows to be joined lie over queries and tiles");
  static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "");
};

__device__ __forceinline__ uint32_t idesc_bf16(uint32_t m, uint32_t n, uint32_t b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// shared-memory descriptor, 128B swizzle, leading and stride byte offsets
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 | static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32 |
         static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_limited(bar, parity, kWaitLimit)); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst_smem, const void* tmap, uint32_t bar, int32_t c0, int32_t c1, int32_t c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ float4 peer_float4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float2 peer_float2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ bool odd_pair(uint32_t u) { return (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u; }      // an infinity or NaN among two bf16
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

// Rows that no request owns, and those of requests that are left out, become zeros (one block).
__device__ void zero_rest(const b200_tree_attn_args& a) {
  bool plain = true;
  for (int s = threadIdx.x; s < a.S; s += blockDim.x) {
    const int rows = a.starts[s + 1] - a.starts[s];
    plain = plain && a.starts[s] >= 0 && rows >= 0 && tree::request_of(a.starts, a.ctx, s, a.T, a.max_blocks, a.max_tree).rows == rows;
  }
  plain = __syncthreads_and(plain);
  const int from = plain && a.S ? a.starts[0] : 0, to = plain && a.S ? a.starts[a.S] : 0;
  for (int t = 0; t < a.T; ++t) {
    bool owned = plain && t >= from && t < to;
    if (owned) { t = to - 1; continue; }
    for (int s = 0; !plain && s < a.S && !owned; ++s) {
      const tree::Request r = tree::request_of(a.starts, a.ctx, s, a.T, a.max_blocks, a.max_tree);
      owned = t >= r.row0 && t < r.row0 + r.rows;
    }
    if (owned) continue;
    uint4* out = reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) + static_cast<size_t>(t) * a.ldo);
    for (int c = threadIdx.x; c < a.q_heads * (kD / 8); c += blockDim.x) out[c] = make_uint4(0, 0, 0, 0);
  }
}

template <int NT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, Shape<NT>::kCtas)
tree_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ b200_tree_attn_args a, float scale_log2, int* error) {
  constexpr int kStages = Shape<NT>::kStages, kWarps = Shape<NT>::kThreads / 32;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t q_s = sbase, k_s = sbase + Shape<NT>::kRing, v_s = k_s + kStages * kTile, bars = sbase + Shape<NT>::kBars;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (kStages + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 * kStages + s); };
  auto v_empty = [&](int s) { return bars + 8u * (3 * kStages + s); };
  auto s_full = [&](int i, int b) { return bars + 8u * (4 * kStages + 2 * i + b); };
  // of every other tile each, as the scores': a warp is up to two tiles ahead of the slowest one of its group
  auto p_ready = [&](int i, int b) { return bars + 8u * (4 * kStages + 4 + 2 * i + b); };
  auto pv_full = [&](int i, int b) { return bars + 8u * (4 * kStages + 8 + 2 * i + b); };
  const uint32_t q_bar = bars + 8u * (4 * kStages + 12), slot = q_bar + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + (slot - sbase));
  volatile uint32_t* odd_values = tmem_slot + 1;
  const int warp = warp_number(), lane = threadIdx.x & 31;

  const int parts = static_cast<int>(gridDim.x), part = static_cast<int>(blockIdx.x);
  const int kvh = blockIdx.y % a.kv_heads, block = blockIdx.y / a.kv_heads, s = blockIdx.z;
  const int group = a.q_heads / a.kv_heads, block_rows = NT * kRows / group;      // tokens of a block
  griddep_enter();
  if (s == a.S) {
    if (part == 0 && blockIdx.y == 0) zero_rest(a);
    return;
  }
  const tree::Request r = tree::request_of(a.starts, a.ctx, s, a.T, a.max_blocks, a.max_tree);
  const int first = block * block_rows, nb = min(block_rows, r.rows - first);      // this block's tokens of the request
  if (nb <= 0) return;
  const int kv_end = r.ctx + (a.masks ? r.rows : first + nb), all_tiles = (kv_end + kKeys - 1) / kKeys;
  // its part of the tiles; parts that find none leave (a cluster barrier does not wait for threads that have ended)
  const int per = max((all_tiles + parts - 1) / parts, 2), active = (all_tiles + per - 1) / per;
  if (part >= active) return;
  const int t_begin = part * per, t_end = min(all_tiles, t_begin + per), tiles = t_end - t_begin;
  const int tiles_q = NT == 2 && nb * group > kRows ? 2 : 1;
  auto warps_of = [&](int i) { return (min(nb * group - i * kRows, kRows) + 31) / 32; };

  if (warp == 0) {
    if (lane == 0) {
      for (int st = 0; st < kStages; ++st) {
        mbar_init(k_full(st), 1); mbar_init(k_empty(st), 1); mbar_init(v_full(st), 1); mbar_init(v_empty(st), 1);
      }
      for (int i = 0; i < tiles_q; ++i)
        for (int b = 0; b < 2; ++b) { mbar_init(s_full(i, b), 1); mbar_init(p_ready(i, b), warps_of(i)); mbar_init(pv_full(i, b), 1); }
      mbar_init(q_bar, 1);
      fence_mbar_init();
      *odd_values = 0;
    }
    __syncwarp();
    tmem_alloc(slot, 256 * NT);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto tm_s = [&](int i, int b) { return tmem + 64u * (2 * i + b); };
  auto tm_o = [&](int i) { return tmem + 128u * NT + 128u * i; };
  bool ok = true;
  float ref = -INFINITY, l = 0.f;      // of a softmax thread's row: what its weights are relative to, in units of log 2, and their sum

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    const bool one = elect_one();
    if (one) mbar_arrive_expect_tx(q_bar, tiles_q * 2 * kQSlab);
    for (int i = 0; i < tiles_q; ++i)
      for (int h = 0; h < 2; ++h)
        if (one) tma_load_3d(q_s + (2 * i + h) * kQSlab, &tm_q, q_bar, 64 * h, kvh * group, r.row0 + first + i * (kRows / group));
    const int pages = (kv_end + 15) >> 4, p_begin = t_begin * 4;
    const int* table = a.block_tables + static_cast<size_t>(s) * a.ld_tables;
    // a page that the cache does not have lies behind its last row, where a load finds zeros
    auto look_up = [&](int base) {
      const int p = base + lane, page = p < pages ? table[p] : -1;
      return page >= 0 && page < a.num_pages ? page : static_cast<int>(a.num_pages);
    };
    const uint64_t hint = gridDim.y > static_cast<unsigned>(a.kv_heads) ? kEvictNormal : kEvictFirst;
    int mine = look_up(p_begin), next = look_up(p_begin + 32);
    for (int it = 0; it < tiles; ++it) {
      if (it && it % 8 == 0) {
        mine = next;
        next = look_up(p_begin + 4 * it + 32);
      }
      const int st = it % kStages, n = min(4, pages - p_begin - 4 * it);
      const uint32_t parity = ((it / kStages) & 1) ^ 1u;
#pragma unroll
      for (int w = 0; w < 2; ++w) {      // keys, then values
        if (!(ok = warp_wait(w ? v_empty(st) : k_empty(st), parity))) break;
        const uint32_t full = w ? v_full(st) : k_full(st), dst = (w ? v_s : k_s) + st * kTile;
        if (one) mbar_arrive_expect_tx(full, n * 4096);
#pragma unroll
        for (int pg = 0; pg < 4; ++pg) {
          const int page = __shfl_sync(0xffffffffu, mine, (4 * it + pg) & 31), row = ((page * 2 + w) * a.kv_heads + kvh) * 16;
          if (pg >= n || !one) continue;
          tma_load_2d(dst + pg * 2048, &tm_kv, full, 0, row, hint);
          tma_load_2d(dst + kSlab + pg * 2048, &tm_kv, full, 64, row, hint);
        }
      }
      if (!ok) {
        // the copies in flight land before the CTA ends
        for (int j = max(0, it - kStages); j <= it; ++j) { warp_wait(k_full(j % kStages), (j / kStages) & 1); warp_wait(v_full(j % kStages), (j / kStages) & 1); }
        break;
      }
    }
    warp_wait(q_bar, 0);
  } else if (warp == kWarps - 1) {
    // ------------------------------------------------------------ products
    const bool one = elect_one();
    const uint32_t id_s = idesc_bf16(kRows, kKeys, 0), id_o = idesc_bf16(kRows, kD, 1);
    const uint64_t q_d = desc_sw128(q_s, 16, 1024), k_d = desc_sw128(k_s, 16, 1024), v_d = desc_sw128(v_s, kSlab, 1024);
    auto scores = [&](int it) {
      const int st = it % kStages;
      if (!warp_wait(k_full(st), (it / kStages) & 1)) return false;
      tc_fence_after();
      if (one) {
        for (int i = 0; i < tiles_q; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) umma_bf16_k64(tm_s(i, it & 1), q_d + (2 * i + h) * (kQSlab >> 4), k_d + st * (kTile >> 4) + h * (kSlab >> 4), id_s, h);
          umma_commit(s_full(i, it & 1));
        }
        umma_commit(k_empty(st));
      }
      __syncwarp();
      return true;
    };
    ok = warp_wait(q_bar, 0) && scores(0);
    for (int it = 0; ok && it < tiles; ++it) {
      // the next scores go to the other buffers, whose readers have handed in their P of the tile before this one
      if (it + 1 < tiles && !(ok = scores(it + 1))) break;
      const int st = it % kStages, kv0 = (t_begin + it) * kKeys;
      if (!(ok = warp_wait(v_full(st), (it / kStages) & 1))) break;
      if (kv0 + kKeys > r.ctx) {
        bool odd = false;
        for (int e = max(0, r.ctx - kv0) * 8 + lane; e < kKeys * 8; e += 32) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4* v = reinterpret_cast<uint4*>(smem + (v_s - sbase) + st * kTile + h * kSlab) + e;      // (a row's pieces in some order)
            if (kv0 + (e >> 3) >= kv_end) *v = make_uint4(0, 0, 0, 0);
            else if (const uint4 x = *v; odd_pair(x.x) || odd_pair(x.y) || odd_pair(x.z) || odd_pair(x.w)) {
              *v = make_uint4(without_odd(x.x), without_odd(x.y), without_odd(x.z), without_odd(x.w));
              odd = true;
            }
          }
        }
        if (odd) *odd_values = 1;
        fence_proxy_async();
        __syncwarp();
      }
      for (int i = 0; i < tiles_q; ++i) {
        if (!(ok = warp_wait(p_ready(i, it & 1), (it >> 1) & 1))) break;
        tc_fence_after();
        if (one) {
          umma_bf16_tmem_k64(tm_o(i), tm_s(i, it & 1), v_d + st * (kTile >> 4), id_o, it > 0);
          umma_commit(pv_full(i, it & 1));
        }
        __syncwarp();
      }
      if (ok && one) umma_commit(v_empty(st));
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax: thread = row (token * group + head)
    const int gi = (warp - 1) >> 2, q = warp & 3, row = gi * kRows + q * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    const bool valid = row < nb * group;
    const int token = first + row / group;
    const int* mask = a.masks && valid ? a.masks + static_cast<size_t>(r.row0 + token) * a.words : nullptr;
    if (gi < tiles_q && gi * kRows + q * 32 < nb * group) {
      for (int it = 0; it < tiles; ++it) {
        const int b = it & 1, kv0 = (t_begin + it) * kKeys;
        if (!(ok = warp_wait(s_full(gi, b), (it >> 1) & 1))) break;
        tc_fence_after();
        uint32_t s0[32], s1[32];
        tmem_ld_32x32(tm_s(gi, b) + lane_off, s0);
        tmem_ld_32x32(tm_s(gi, b) + lane_off + 32, s1);
        tmem_ld_wait();
        if (kv0 + kKeys > r.ctx) {
          const uint32_t m0 = valid ? seen_bits(mask, a.words, token, r.rows, kv0 - r.ctx) : 0u, m1 = valid ? seen_bits(mask, a.words, token, r.rows, kv0 + 32 - r.ctx) : 0u;
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
        auto weight = [&](uint32_t u) { return exp2_ftz(fmaf(__uint_as_float(u), scale_log2, -mu)); };
        float ps = 0.f;
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const float p0 = weight(s0[c]), p1 = weight(s0[c + 1]), p2 = weight(s1[c]), p3 = weight(s1[c + 1]);
          ps += (p0 + p1) + (p2 + p3);
          pk[c >> 1] = pack_bf16x2(p0, p1);
          pk[16 + (c >> 1)] = pack_bf16x2(p2, p3);
        }
        l = l * alpha + ps;
        // P in place of the scores: what read this buffer's last P went ahead of them.  Where some row of the warp moved its maximum, its output so
        // far is scaled once the previous tile's product has landed.
        tmem_st_32x32(tm_s(gi, b) + lane_off, pk);
        if (it > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
          if (!(ok = warp_wait(pv_full(gi, b ^ 1), ((it - 1) >> 1) & 1))) break;
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < kD; c0 += 32) {
            uint32_t v[32];
            tmem_ld_32x32(tm_o(gi) + lane_off + c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * alpha);
            tmem_st_32x32(tm_o(gi) + lane_off + c0, v);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(gi, b));
      }
      if (ok) ok = warp_wait(pv_full(gi, (tiles - 1) & 1), ((tiles - 1) >> 1) & 1);
    }
  }
  if (!ok) *reinterpret_cast<volatile int*>(error) = 1;
  ok = __syncthreads_and(ok);      // every product and copy has landed: queries and tiles may be written over
  tc_fence_after();

  // ------------------------------------------------------------ results
  const int rows = nb * group;
  float* joined = reinterpret_cast<float*>(smem);                       // [rows][kLd], then [rows] of maximum and sum
  float2* state = reinterpret_cast<float2*>(joined + NT * kRows * kLd);
  if (ok && warp >= 1 && warp < kWarps - 1) {
    const int gi = (warp - 1) >> 2, q = warp & 3, row = gi * kRows + q * 32 + lane, token = first + row / group;
    if (gi * kRows + q * 32 < rows) {
      const bool valid = row < rows;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      bf16* dst = static_cast<bf16*>(a.out) + static_cast<size_t>(r.row0 + token) * a.ldo + (kvh * group + row % group) * kD;
      const int* mask = a.masks && valid ? a.masks + static_cast<size_t>(r.row0 + token) * a.words : nullptr;
#pragma unroll
      for (int c0 = 0; c0 < kD; c0 += 32) {
        uint32_t v[32];
        tmem_ld_32x32(tm_o(gi) + (static_cast<uint32_t>(q * 32) << 16) + c0, v);
        tmem_ld_wait();
        if (!valid) continue;
        if (*odd_values) {
          // infinities and NaN of the drafts that this row sees, which stayed out of the products
          const int* table = a.block_tables + static_cast<size_t>(s) * a.ld_tables;
          for (int p = max(r.ctx, t_begin * kKeys); p < min(kv_end, t_end * kKeys); ++p) {
            if (!(seen_bits(mask, a.words, token, r.rows, p - r.ctx) & 1)) continue;
            const long long at = tree::cache_row(table, p, a.num_pages);
            if (at < 0) continue;
            const bf16* value = static_cast<const bf16*>(a.kv_layer) + ((((at >> 4) * 2 + 1) * a.kv_heads + kvh) * 16 + (at & 15)) * kD + c0;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float x = __bfloat162float(value[c]);
              if (!isfinite(x)) v[c] = __float_as_uint(__uint_as_float(v[c]) + x);
            }
          }
        }
        if (active == 1) {
#pragma unroll
          for (int c = 0; c < 32; c += 8)
            *reinterpret_cast<uint4*>(dst + c0 + c) =
                make_uint4(pack_bf16x2(__uint_as_float(v[c]) * inv, __uint_as_float(v[c + 1]) * inv), pack_bf16x2(__uint_as_float(v[c + 2]) * inv, __uint_as_float(v[c + 3]) * inv),
                           pack_bf16x2(__uint_as_float(v[c + 4]) * inv, __uint_as_float(v[c + 5]) * inv), pack_bf16x2(__uint_as_float(v[c + 6]) * inv, __uint_as_float(v[c + 7]) * inv));
        } else {
#pragma unroll
          for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(joined + row * kLd + c0 + c) = make_uint4(v[c], v[c + 1], v[c + 2], v[c + 3]);
        }
      }
      if (active > 1 && valid) state[row] = make_float2(ref, l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 256 * NT);
  }
  if (active == 1) return;
  // the parts' rows, each by a warp of one of the CTAs: sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p
  __syncwarp();
  cluster_sync_all();
  if (ok) {
    const uint32_t at_joined = smem_u32(joined), at_state = smem_u32(state);
    for (int row = part + active * warp; row < rows; row += active * kWarps) {
      float2 st[kMostParts];
      float m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int p = 0; p < kMostParts; ++p)
        if (p < active) {
          st[p] = peer_float2(mapa_u32(at_state + row * 8, p));
          m = fmaxf(m, st[p].x);
        }
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < kMostParts; ++p)
        if (p < active) {
          const float w = st[p].x == -INFINITY && st[p].y == 0.f ? 0.f : exp2f(st[p].x - m);      // (a row that sees nothing of this part)
          const float4 x = peer_float4(mapa_u32(at_joined + (row * kLd + lane * 4) * 4, p));
          sum = fmaf(st[p].y, w, sum);
          if (w != 0.f) o = make_float4(fmaf(x.x, w, o.x), fmaf(x.y, w, o.y), fmaf(x.z, w, o.z), fmaf(x.w, w, o.w));
        }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint2 y;
      y.x = pack_bf16x2(o.x * inv, o.y * inv);
      y.y = pack_bf16x2(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + static_cast<size_t>(r.row0 + first + row / group) * a.ldo + (kvh * group + row % group) * kD + lane * 4) = y;
    }
  }
  __syncwarp();
  cluster_sync_all();      // no CTA leaves while its rows are read
}

template <int NT>
int launch(const b200_tree_attn_args& a, int* error, cudaStream_t st) {
  const int group = a.q_heads / a.kv_heads;
  CUtensorMap tm_q, tm_kv;
  if (int rc = tmap_encode_bf16_3d(&tm_q, a.q, kD, a.q_heads, a.T, kD, a.ldq, 64, group, kRows / group)) return rc;
  if (int rc = tmap_encode_bf16_2d(&tm_kv, a.kv_layer, static_cast<uint64_t>(a.num_pages) * 2 * a.kv_heads * 16, kD, kD, 16, 64, 1)) return rc;
  const auto kernel = tree_attn_kernel<NT>;
  static std::atomic<unsigned long long> attr_done{0};
  if (!ensure_dynamic_smem(kernel, Shape<NT>::kSmem, &attr_done)) return -3;
  const long long blocks = static_cast<long long>((std::min(a.max_tree, a.T) * static_cast<long long>(group) + NT * kRows - 1) / (NT * kRows)) * a.kv_heads;
  if (blocks > 65535) return -1;
  // parts of a context: enough CTAs for the SMs, each with four tiles at least where the contexts are as long as that
  const int most = a.max_ctx > 0 ? std::min(a.max_ctx, a.max_blocks * tree::kPage) : a.max_blocks * tree::kPage;
  const int tiles = most / kKeys + 1;
  int parts = 1;
  while (parts < kMostParts && parts * 8 <= tiles && blocks * a.S * parts < 4ll * Shape<NT>::kCtas * sm_count()) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, static_cast<unsigned>(blocks), a.S + (a.zero_rest ? 1 : 0));
  cfg.blockDim = dim3(Shape<NT>::kThreads);
  cfg.dynamicSmemBytes = Shape<NT>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, tm_q, tm_kv, a, a.scale * 1.4426950408889634f, error) == cudaSuccess ? 0 : -2;
}

}  // namespace

int paged_attention_tree(const b200_tree_attn_args& a, int* error, cudaStream_t st) {
  const int group = a.q_heads / a.kv_heads;
  return static_cast<long long>(std::min(a.max_tree, a.T)) * group <= kRows ? launch<1>(a, error, st) : launch<2>(a, error, st);
}

}  // namespace b200
