// Attention of parts of many rows, on the 5th-generation tensor cores: a group's rows over the pages that it shares, and the own keys of requests with long chains
// (shared_attention.cu has the parts, the joining and what parts of few rows take).
//
// An item is a part's key head and up to 256 of its rows (row = token * group + head).  Every step forms two tiles of scores, 128 rows by 128 keys: of two row tiles that share 128 keys, or
// where there are no more than 128 rows of one row tile and 256 keys.  All items' steps one behind the other are cut into as many equal ranges as there are CTAs of this kind, one an SM, and
// a CTA walks its range without a gap:
//   a warp looks pages up and loads by TMA, 128-byte swizzle: queries, and tiles of 128 keys or values into a ring of four;
//   a warp issues tcgen05.mma: S_g = Q K^T and O_g += P_g V (M = N = 128), P_g in TMEM over its scores: the next scores of one tile are formed under the other's softmax;
//   two groups of four warps (thread = row) do the softmax in fp32, base 2; a warp whose rows nobody owns only keeps step.
// The scores of a step come behind the products with the last step's values in the order of their issue, so a tile whose scores are there has its O at rest: no other wait stands in front of its rescaling.
// Weights are relative to the row's largest score so far, rounded to bf16 (by up to 2^-8 of each) and divided by the sum of the rounded ones, as in narrow CTAs: what all values have in common has no
// part of the rounding.  The sum of the unrounded weights left up to 2^-8 of the output there and was cheaper: 128 rows behind 2048 tokens 49.3 us, not 50.9, 4 groups of 160 rows behind 8000 57.3, not 61.8,
// the questions below 256, not 265.  (An older maximum, kept until it grew by a factor of two, spares rescalings of O: 263 for the questions; nothing elsewhere.)
// Only steps that reach behind what every row sees are masked.  There the products' warp also clears what must not meet a weight of zero: values behind the last key, and infinities and NaN
// among values that some row does not see, which the rows that see them add at the end by themselves.
// Every wait has a limit; a CTA that gives up sets an error mark and still meets at the end.
// 2 x 24 questions of up to 32 tokens about 16001, 211 GFLOP: 265 us (285 under the power cap), 0.80 PFLOP/s, 50 % of what a large product reaches.  A CTA has some 95 steps of two tiles in 391,000 cycles,
// 4100 a step: tensor cores and the exponentials' unit are busy for 45 %, issue slots for 42 %.  What bounds it is a tile's chain (scores, load, maximum, 128 exponentials a thread, weights out, products):
// with the sum of the unrounded weights, 255 us, it took 221 without loads and 219 without the softmax; half tiles of 64 keys with scores ahead of them 300, sixteen softmax warps 287, another order of the
// exponentials' instructions the same.  The sum behind the weights' way out, under the products, is no faster (265).
#pragma once
#include "shared_attention.cuh"

namespace b200 {
namespace shared_attn {
namespace wide {

constexpr int kTileRows = 128, kKeys = 128;                         // of a tile of scores
constexpr int kSlab = 128 * 128, kTile = 2 * kSlab;                 // bytes: 64 columns of 128 rows, a tile
constexpr int kThreads = 384, kRing = 4;                                            // tiles of keys and values.  Warps 0 to 3 and 4 to 7: softmax, 8: loads, 9: products
constexpr int kLeast = 4;                                           // steps of a range at least: its rows leave as 132 KB, as much as four tiles

// shared memory: queries, ring, 2 KB a softmax warp for its way out, barriers
constexpr int kRingAt = 2 * kTile, kStageAt = kRingAt + kRing * kTile, kBars = kStageAt + 8 * 2048, kSmem = 1024 + kBars + 256;

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The registers that a warpgroup's threads keep of a launch with 168 each: 2 * 216 + 72 = 3 * 168
template <int kRegs>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

// An item's steps of a range, as the loads leave them for the other roles
struct Piece {
  int take;                  // steps
  int key, end, see;         // first key, keys behind the last, and behind the last that the block's token 0 sees; token i sees i more
  int rows, row0, kvh, table;
  short tall, whole, begins, own, joined, last;      // two row tiles; all of the item, its beginning; a request's own keys, behind shared ones; the range's last
};
constexpr int kPieces = 4;      // the loads are never that many items ahead: an item has two tiles at least, and the ring four

// A range's steps, one behind the other
struct Steps {
  Piece x;
  int j, item, seq;      // step of the item, items so far, tiles of the ring so far
  bool more;
  __device__ __forceinline__ int key(int g) const { return x.key + j * (x.tall ? kKeys : 2 * kKeys) + (x.tall ? 0 : g * kKeys); }      // the first of a tile of scores
  __device__ __forceinline__ bool active(int g) const { return g == 0 || x.tall || key(1) < x.end; }
  __device__ __forceinline__ int tiles() const { return x.tall ? 1 : 1 + active(1); }                   // of keys, and of values, of this step
  __device__ __forceinline__ int key_tile(int g) const { return seq + (x.tall ? 0 : g); }
  __device__ __forceinline__ int value_tile(int g) const { return seq + (x.tall ? 1 : tiles() + g); }
  __device__ __forceinline__ bool last() const { return j + 1 == x.take; }
  // whether the item's piece has come
  __device__ __forceinline__ bool open(const Piece* pieces, uint32_t bars) {
    if (!warp_wait(bars + 8u * (item % kPieces), (item / kPieces) & 1)) return false;
    x = pieces[item % kPieces];
    j = 0;
    return true;
  }
  __device__ __forceinline__ bool begin(const Piece* pieces, uint32_t bars) {
    item = seq = 0;
    more = true;
    return open(pieces, bars);
  }
  __device__ __forceinline__ bool next(const Piece* pieces, uint32_t bars) {
    seq += 2 * tiles();
    if (++j < x.take) return true;
    if (x.last) { more = false; return true; }
    ++item;
    return open(pieces, bars);
  }
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
  const b200_shared_attn_args& a;
  uint8_t* stage;
  int rows, row0, lane, group, shift;      // the item's rows, the warp's first one
  long long first;                         // the item's first row of the step
  int kvh, table;
  float* part;                             // fp32 rows with their maximum and sum: the range's slot, or null for the rows of all, from `all` on
  float* all;
  bool last;                               // normalised rows to the output
  int odd_from, odd_to;                    // keys whose odd values this thread's row adds

  __device__ __forceinline__ float* row_at(int to) const {
    return part ? part + static_cast<size_t>(to) * kLd : all + ((first + (to >> shift)) * a.q_heads + kvh * group + (to & (group - 1))) * kLd;
  }
  // columns c0 .. c1 of fa times the output at oa in TMEM, with `two` and fb times that at ob; m in units of log 2
  __device__ __forceinline__ void write(int c0, int c1, uint32_t oa, float fa, bool two, uint32_t ob, float fb, float m, float sum) const {
    const int row = row0 + lane;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    // two rows are a line of 128 bytes, pieces of 16 bytes in an order that leaves no bank twice
    auto piece = [&](int r, int k) { return reinterpret_cast<uint4*>(stage + (r >> 1) * 128 + ((((r & 1) * 4 + k) ^ ((r >> 1) & 7)) << 4)); };
#pragma unroll 1
    for (int c = c0; c < c1; c += 32) {
      uint32_t v[32];
      tmem_ld_32x32(oa + c, v);
      tmem_ld_wait();
      if (two) {
        uint32_t u[32];
        tmem_ld_32x32(ob + c, u);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          v[i] = __float_as_uint((fa == 0.f ? 0.f : __uint_as_float(v[i]) * fa) + (fb == 0.f ? 0.f : __uint_as_float(u[i]) * fb));
      }
      if (odd_from < odd_to && row < rows) {
        uint32_t y[32];
        for (int i = 0; i < 32; ++i) y[i] = v[i];
        add_odd(a, table, kvh, odd_from, odd_to, c, y);
        for (int i = 0; i < 32; ++i) v[i] = y[i];
      }
      auto leave = [&](int to_column) {      // what lies there, 64 bytes a row
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2), k = lane & 3, to = row0 + r;
          const uint4 x = *piece(r, k);
          if (to >= rows) continue;
          if (last)
            *reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) + (first + (to >> shift)) * a.ldo + (kvh * group + (to & (group - 1))) * kD + to_column + 8 * k) = x;
          else
            *reinterpret_cast<uint4*>(row_at(to) + to_column + 4 * k) = x;
        }
        __syncwarp();
      };
      if (last) {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          *piece(lane, i / 8) =
              make_uint4(pack_bf16x2(__uint_as_float(v[i]) * inv, __uint_as_float(v[i + 1]) * inv), pack_bf16x2(__uint_as_float(v[i + 2]) * inv, __uint_as_float(v[i + 3]) * inv),
                         pack_bf16x2(__uint_as_float(v[i + 4]) * inv, __uint_as_float(v[i + 5]) * inv), pack_bf16x2(__uint_as_float(v[i + 6]) * inv, __uint_as_float(v[i + 7]) * inv));
        leave(c);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) *piece(lane, i / 4) = make_uint4(v[16 * h + i], v[16 * h + i + 1], v[16 * h + i + 2], v[16 * h + i + 3]);
          leave(c + 16 * h);
        }
      }
    }
    if (!last && c0 == 0 && row < rows) *reinterpret_cast<float2*>(row_at(row) + kD) = make_float2(m, sum);
  }
};

struct Shared {
  float2 states[2][kTileRows];      // maximum and sum of each group's rows, where two groups have the same ones
  Piece pieces[kPieces];
};

// The range of CTA `cta` of this half, which begins and ends as `range` and `where` have it
__device__ __forceinline__ void walk(const CUtensorMap& tm_q, const CUtensorMap& tm_kv, const b200_shared_attn_args& a, const Sizes& sizes, float scale_log2, int* error, uint8_t* smem, Shared& shared,
                                     const Lengths& n, const tree::Ranges& ranges, int cta, const int* s_range, const int (*s_where)[4]) {
  Piece* pieces = shared.pieces;
  auto& states = shared.states;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t q_s = sbase, ring = sbase + kRingAt, bars = sbase + kBars;
  auto full = [&](int n) { return bars + 8u * (n % kRing); };
  auto empty = [&](int n) { return bars + 8u * (kRing + n % kRing); };
  auto round = [&](int n) { return static_cast<uint32_t>(n / kRing) & 1u; };
  auto s_full = [&](int g) { return bars + 8u * (8 + g); };
  auto p_ready = [&](int g, int h) { return bars + 8u * (10 + 2 * g + h); };      // halves of 64 keys
  auto pv_full = [&](int g) { return bars + 8u * (14 + g); };
  auto meet = [&](int q) { return bars + 8u * (16 + q); };      // of the two warps of a quarter of the lanes
  const uint32_t q_full = bars + 8u * 20, q_empty = bars + 8u * 21, piece_full = bars + 8u * 22, slot = bars + 8u * 26;
  static_assert(kRing == 4 && kPieces == 4 && 8 * 26 + 8 + 4 * kPieces <= 256, "");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + (slot - sbase));
  volatile int* odd_item = reinterpret_cast<volatile int*>(tmem_slot + 2);      // [kPieces]: the last item of each piece's place with infinities or NaN among values that some row does not see.
  // (The products may be two items ahead of a group without scores in the one between: item i + 2's marks may be made before that group has looked at item i's.  Its end is where both groups meet,
  // in front of any product of item i + 3.)
  const int warp = warp_number(), lane = threadIdx.x & 31, tid = threadIdx.x;

  const int group = a.q_heads / a.kv_heads, shift = __ffs(group) - 1;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kRing; ++s) {
        mbar_init(full(s), 1);
        mbar_init(empty(s), 1);
      }
      for (int g = 0; g < 2; ++g) {
        mbar_init(s_full(g), 1); mbar_init(p_ready(g, 0), 4); mbar_init(p_ready(g, 1), 4); mbar_init(pv_full(g), 1);
      }
      for (int q = 0; q < 4; ++q) {
        mbar_init(meet(q), 2);
        mbar_init(piece_full + 8u * q, 1);
      }
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      fence_mbar_init();
      for (int i = 0; i < kPieces; ++i) odd_item[i] = -1;
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_kv);
    }
    __syncwarp();
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
  const Items I(0, group);
  bool ok = true;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto tm_s = [&](int g) { return tmem + 128u * g; };
  auto tm_o = [&](int g) { return tmem + 256u + 128u * g; };

  const bool some_work = s_range[1] > s_range[0];
  if (warp >= 8) {
    fewer_registers<72>();
    if (some_work && warp == 8) {
      // ------------------------------------------------------------ loads
      const bool one = elect_one();
      const int bt = I.bt;
      Item it;
      it.u = s_where[0][0]; it.kvh = s_where[0][1]; it.block = s_where[0][2];
      it.p = I.part(n, it.u);
      it.fill(I);
      int t0 = max(0, s_range[0] - s_where[0][3] - tree::kItem), rest = s_range[1] - s_range[0];
      if (t0 == it.units) {      // the range begins where the item in front of it ends
        t0 = 0;
        it.next(n, I, a.kv_heads);
      }
      Space space = space_of(a, sizes);
      int seq = 0, item = 0, queries = 0;      // tiles issued, items, items whose queries are on their way
      for (;; ++item) {
        const int take = tree::take_of(t0, it.units, &rest);
        const bool tall = 2 * it.nb > bt, whole = t0 == 0 && take == it.units;
        const int unit = tall ? kKeys : 2 * kKeys, pages = (it.k1 - it.p.k0 + 15) >> 4, p_begin = t0 * (unit / 16), row0 = it.p.row0 + it.first;
        if (lane == 0) {
          Piece x;
          x.take = take;
          x.key = it.p.k0 + 16 * p_begin;
          x.end = it.k1;
          x.see = it.p.all ? it.k1 : it.p.ctx + it.first + 1;
          x.rows = it.nb * group;
          x.row0 = row0;
          x.kvh = it.kvh;
          x.table = it.p.table;
          x.tall = tall;
          x.whole = whole;
          x.begins = t0 == 0;
          x.own = !it.p.all;
          x.joined = it.p.k0 > 0;
          x.last = rest <= 0;
          pieces[item % kPieces] = x;
          mbar_arrive(piece_full + 8u * (item % kPieces));
        }
        __syncwarp();
        const int* table = a.block_tables + static_cast<size_t>(it.p.table) * a.ld_tables + it.p.k0 / 16;
        // 32 pages at a time: the first row of a page's keys; a page that the cache does not have lies behind its last row, where a load finds zeros
        auto look_up = [&](int p) {
          const int page = p < pages ? table[p] : -1;
          return ((page >= 0 && page < a.num_pages ? page : static_cast<int>(a.num_pages)) * 2 * a.kv_heads + it.kvh) * 16;
        };
        const uint64_t hint = it.p.rows > bt ? kEvictNormal : kEvictFirst;
        int base = p_begin, mine = look_up(base + lane), next = look_up(base + 32 + lane);
        for (int j = 0; ok && j < take; ++j) {
          const int first = p_begin + j * (unit / 16), tiles = tall || first + 8 >= pages ? 1 : 2;
          if (first + 8 * tiles > base + 32) {
            base += 32;
            mine = next;
            next = look_up(base + 32 + lane);
          }
          for (int x = 0; x < 2 * tiles; ++x, ++seq) {
            const bool values = x >= tiles;
            if (x == tiles && j == 0) {      // queries, behind the first keys, which need not wait for the last item's scores
              if (!(ok = warp_wait(q_empty, (item & 1) ^ 1u))) break;
              if (one) {
                mbar_arrive_expect_tx(q_full, tall ? 2 * kTile : kTile);
                for (int g = 0; g < (tall ? 2 : 1); ++g)
                  for (int h = 0; h < 2; ++h) tma_load_3d(q_s + g * kTile + h * kSlab, &tm_q, q_full, 64 * h, it.kvh * group, row0 + g * (kTileRows / group));
              }
              __syncwarp();
              queries = item + 1;
            }
            const int p0 = first - base + 8 * (values ? x - tiles : x), count = min(8, pages - base - p0);
            if (!(ok = warp_wait(empty(seq), round(seq) ^ 1u))) break;
            if (one) mbar_arrive_expect_tx(full(seq), count * 4096);
            __syncwarp();
            const uint32_t dst = ring + (seq % kRing) * kTile;
            int row[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) row[p] = __shfl_sync(0xffffffffu, mine, (p0 + p) & 31) + (values ? 16 * a.kv_heads : 0);
            if (one) {
#pragma unroll
              for (int p = 0; p < 8; ++p) {
                if (p >= count) break;
                tma_load_2d(dst + p * 2048, &tm_kv, full(seq), 0, row[p], hint);
                tma_load_2d(dst + kSlab + p * 2048, &tm_kv, full(seq), 64, row[p], hint);
              }
            }
            __syncwarp();
          }
        }
        if (!ok) break;
        if (t0 == 0) {      // where the item's rows are: their tokens', 32 at a time
          const int parts = whole ? 0 : ranges.parts(cta, s_range[1] - take, it.units), flags = it.p.k0 > 0 ? kJoined : 0;
          for (int i = lane; i < it.nb; i += 32)
            space.places[(static_cast<size_t>(!it.p.all) * a.T + row0 + i) * a.kv_heads + it.kvh] = {2 * cta + 1, parts, i << shift, flags};
        }
        if (rest <= 0) break;
        t0 = 0;
        it.next(n, I, a.kv_heads);
      }
      // the copies in flight land before the CTA ends, also where it gives up
      if (queries) warp_wait(q_full, (queries - 1) & 1);
      for (int k = max(0, seq - kRing); k < seq; ++k) warp_wait(full(k), round(k));
    } else if (some_work && warp == 9) {
      // ------------------------------------------------------------ products: scores run a step ahead
      const bool one = elect_one();
      const uint32_t id_s = idesc_bf16(kTileRows, kKeys, 0), id_o = idesc_bf16(kTileRows, kD, 1);
      const uint64_t q_d = desc_sw128(q_s, 16, 1024), k_d = desc_sw128(ring, 16, 1024), v_d = desc_sw128(ring, kSlab, 1024);
      Steps w, v;      // w: scores, v: outputs
      ok = w.begin(pieces, piece_full) && v.begin(pieces, piece_full);
      int steps[2] = {0, 0}, formed[2] = {0, 0};                             // of outputs, of scores
      auto scores = [&](int g) {
        if (!ok || !w.active(g)) return;
        const int s = w.key_tile(g), at = s % kRing;
        if (!(ok = (w.j > 0 || g > 0 || warp_wait(q_full, w.item & 1)) && warp_wait(full(s), round(s)))) return;
        tc_fence_after();
        if (one) {
          const uint64_t q = q_d + (w.x.tall ? g * (kTile >> 4) : 0);
#pragma unroll
          for (int h = 0; h < 2; ++h) umma_bf16_k64(tm_s(g), q + h * (kSlab >> 4), k_d + at * (kTile >> 4) + h * (kSlab >> 4), id_s, h);
          umma_commit(s_full(g));
          if (!w.x.tall || g == 1) umma_commit(empty(s));
          if (w.last() && !(g == 0 && w.active(1))) umma_commit(q_empty);
        }
        ++formed[g];
        __syncwarp();
      };
      auto outputs = [&](int g) {
        if (!ok || !v.active(g)) return;
        const int s = v.value_tile(g), at = s % kRing, kv0 = v.key(g);
        if (!(ok = warp_wait(full(s), round(s)))) return;
        if (kv0 + kKeys > v.x.see && (g == 0 || !v.x.tall)) {      // (row tiles that share it find it cleared)
          bool odd = false;
          const int from = min(kKeys, max(0, v.x.see - kv0)), end = min(kKeys, v.x.end - kv0);      // the tile's values that some row does not see
          for (int h = 0; h < 2; ++h) {
            uint4* x = reinterpret_cast<uint4*>(smem + kRingAt + at * kTile + h * kSlab);      // (a row's pieces in some order)
            for (int e = from * 8 + lane; e < end * 8; e += 32) {
              const uint4 was = x[e], y = make_uint4(without_odd(was.x), without_odd(was.y), without_odd(was.z), without_odd(was.w));
              if (y.x != was.x || y.y != was.y || y.z != was.z || y.w != was.w) {
                odd = true;
                x[e] = y;
              }
            }
            for (int e = end * 8 + lane; e < kKeys * 8; e += 32) x[e] = make_uint4(0, 0, 0, 0);
          }
          if (odd) odd_item[v.item % kPieces] = v.item;
          __threadfence_block();
          fence_proxy_async();
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!(ok = warp_wait(p_ready(g, h), steps[g] & 1))) return;
          tc_fence_after();
          if (one) umma_bf16_tmem_k64(tm_o(g), tm_s(g) + 32 * h, v_d + at * (kTile >> 4) + 512 * h, id_o, h > 0 || v.j > 0);
          __syncwarp();
        }
        if (one) {
          umma_commit(pv_full(g));
          if (!v.x.tall || g == 1) umma_commit(empty(s));
        }
        ++steps[g];
        __syncwarp();
      };
      scores(0);
      scores(1);
      while (ok && v.more) {
        if (!(ok = w.next(pieces, piece_full))) break;
        outputs(0);
        if (w.more && w.j > 0) scores(0);
        outputs(1);
        if (w.more && w.j > 0) scores(1);
        else if (w.more) {      // another item, whose queries may still be on their way
          scores(0);
          scores(1);
        }
        ok = ok && v.next(pieces, piece_full);
      }
      if (!ok)      // no product is under way when tensor memory is given back
        for (int g = 0; g < 2; ++g) {
          if (formed[g]) warp_wait(s_full(g), (formed[g] - 1) & 1);
          if (steps[g]) warp_wait(pv_full(g), (steps[g] - 1) & 1);
        }
    }
  } else {
    more_registers<216>();
    if (some_work) {
      // ------------------------------------------------------------ softmax: thread = row (token * group + head) of its group's tile
      const int g = warp >> 2, q = warp & 3;      // the quarter of the lanes that this warp may access
      const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16, tm = tm_s(g) + lane_off;
      int steps[2] = {0, 0}, meetings = 0;
      auto met = [&] {      // with the other group's warp of the same lanes
        __syncwarp();
        if (lane == 0) mbar_arrive(meet(q));
        return warp_wait(meet(q), meetings++ & 1);
      };
      float ref = -INFINITY, l = 0.f;      // what the row's weights are relative to, in units of log 2, and their sum
      Steps w;
      ok = w.begin(pieces, piece_full);
      for (; ok && w.more; ok = ok && w.next(pieces, piece_full)) {
        const bool tall = w.x.tall;
        const int row0 = (tall ? g * kTileRows : 0) + q * 32, row = row0 + lane, rows = w.x.rows, see = w.x.see;
        const bool valid = row < rows, some = row0 < rows;      // this warp has rows
        const int limit = valid ? min(see + (row >> shift), w.x.end) : 0;
        if (w.j == 0) {
          ref = -INFINITY;
          l = 0.f;
        }
        if (w.active(g)) {
          const int kv0 = w.key(g);
          if (!(ok = warp_wait(s_full(g), steps[g] & 1))) break;
          if (some) {
            tc_fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld_32x32(tm + 32 * c, s[c]);
            tmem_ld_wait();
            if (kv0 + kKeys > see) {
              const int seen = limit - kv0;
#pragma unroll
              for (int i = 0; i < kKeys; ++i)
                if (i >= seen) s[i >> 5][i & 31] = 0xff800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 2)
#pragma unroll
              for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2;
            float alpha = 1.f;
            if (top > ref) {
              alpha = exp2_ftz(ref - top);
              ref = top;
            }
            if (w.j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
              for (int c0 = 0; c0 < kD; c0 += 32) {
                uint32_t v[32];
                tmem_ld_32x32(tm_o(g) + lane_off + c0, v);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * alpha);
                tmem_st_32x32(tm_o(g) + lane_off + c0, v);
              }
            }
            const float mu = ref == -INFINITY ? 0.f : ref;
            const uint64_t scale2 = pair_of(scale_log2, scale_log2), less2 = pair_of(-mu, -mu);
            uint64_t ps[2] = {0, 0};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t pk[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const int c = 2 * h + (i >> 4), e = 2 * (i & 15);
                const float2 t = floats_of(fma_pair(pair_of(s[c][e], s[c][e + 1]), scale2, less2));
                // the sum is that of the rounded weights
                pk[i] = pack_bf16x2(exp2_ftz(t.x), exp2_ftz(t.y));
                ps[i & 1] = add_pair(ps[i & 1], pair_of(pk[i] << 16, pk[i] & 0xffff0000u));
              }
              tmem_st_32x32(tm + 32 * h, pk);      // P in place of the scores
              if (h == 0) {      // the products with the first half's values may begin
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(g, 0));
              }
            }
            const float2 p0 = floats_of(ps[0]), p1 = floats_of(ps[1]);
            l = l * alpha + ((p0.x + p0.y) + (p1.x + p1.y));
            tmem_st_wait();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) {
            if (!some) mbar_arrive(p_ready(g, 0));
            mbar_arrive(p_ready(g, 1));
          }
        }
        steps[0] += w.active(0);
        steps[1] += w.active(1);
        if (!w.last()) continue;
        // ---- the item's rows
        const Space space = space_of(a, sizes);
        const int begin = w.x.key, end = begin + w.x.take * (tall ? kKeys : 2 * kKeys);
        // a part without the item's beginning is the range's first
        Rows out{a, smem + kStageAt + warp * 2048, rows, row0, lane, group, shift, w.x.row0, w.x.kvh, w.x.table,
                 w.x.whole ? nullptr : space.wide + static_cast<size_t>(2 * cta + w.x.begins) * kWideRows * kLd, space.rows + (w.x.own ? static_cast<size_t>(a.T) * a.q_heads * kLd : 0),
                 w.x.whole && w.x.own && !w.x.joined, 0, 0};
        if (!(ok = warp_wait(pv_full(g), (steps[g] - 1) & 1))) break;
        auto odd = [&] {
          if (odd_item[w.item % kPieces] != w.item) return;
          out.odd_from = max(see, begin);
          out.odd_to = min(limit, end);
        };
        if (tall) {
          tc_fence_after();
          odd();
          if (some) out.write(0, kD, tm_o(g) + lane_off, 1.f, false, 0, 0.f, ref, l);
        } else {
          // both groups have the rows: each writes half of their columns
          states[g][row] = make_float2(ref, l);
          if (!(ok = met() && warp_wait(pv_full(g ^ 1), (steps[g ^ 1] - 1) & 1))) break;
          tc_fence_after();
          odd();
          const float2 x = states[0][row], y = states[1][row];
          const float m = fmaxf(x.x, y.x), base = m == -INFINITY ? 0.f : m, fa = exp2f(x.x - base), fb = exp2f(y.x - base);
          const float sum = (fa == 0.f && x.y == x.y ? 0.f : x.y * fa) + (fb == 0.f && y.y == y.y ? 0.f : y.y * fb);
          if (some) out.write(g * 64, g * 64 + 64, tm_o(0) + lane_off, fa, true, tm_o(1) + lane_off, fb, m, sum);
          tc_fence_before();
          if (!(ok = met())) break;      // the other one has read this one's
        }
        tc_fence_before();
      }
    }
  }
  if (!ok) *reinterpret_cast<volatile int*>(error) = 1;
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace wide
}  // namespace shared_attn
}  // namespace b200
