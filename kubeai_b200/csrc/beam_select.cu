// The best candidates over a request's beams and the vocabulary.
//
//   c(b, v) = score_b + x_bv - m_b - log sum_w exp(x_bw - m_b)        m_b = max_w x_bw
//
// A row's best candidates by c are its best by x, which needs no rounding, so one pass over the logits takes them by x, together with the sum; c, which decides between beams, is
// made in 64 bits for a few hundred candidates.
// First kernel: a row is cut into parts of at most 16384 bf16 (8192 fp32) logits, a CTA each, that come into shared memory by a bulk copy, six CTAs an SM.  A lower bound of the k-th largest value that
// few values besides the k best reach: of every warp the r-th largest of its lanes' maxima (r = k / 4), and of those the fourth largest, as four warps have r lanes each that reach it.  What does goes
// to a list, where each one's place is the number of better ones.  Where more reach it than the list holds, the k-th value and the last token that still belongs are found bit by bit over all values, some
// 50 passes.  So it is for rows of equal values, and for any values where a part has too few for four warps with r lanes each: rows of 257 to 770 (k = 2) or 905 (k = 64) bf16, 257 to 385 or 453 fp32
// (64 requests of 8 beams, k = 16: 500 bf16 43.8 us, 1024 19.3; 400 fp32 34.1, 512 18.8), or parts of which a mask leaves a few hundred neighbours.
// The sum's large terms, those of the list, are taken in 64 bits, the others in 32: what an fp32 sum loses of the large ones would decide between beams whose
// candidates lie close together.  What it loses of the others is less than 2^-18 of the sum (2^-16 where the values are counted), and was 2^-22.5 at most.
// Second kernel, a CTA a request: a beam's candidates come out of its parts' lists one by one, a warp a beam; a candidate's place among those of all beams is its place in its own list and, by bisection,
// in every other.
// 64 requests of 8 beams, 128256 bf16 logits a row: 131 MB, 45.9 us, 36 of them the first kernel's (3.6 TB/s).  Its instructions bound it: 1230 for 128 logits a lane, 530 of them maxima and sum, the
// others the bound, list and places of a part; its four warps a CTA leave half the issue slots empty, and eight of half the logits each took 50 % more instructions (48 us).  Parts of twice the size
// with three CTAs an SM 48.4, one and a half times 49.3 to 53.  The second kernel's 10 us are its chain: heads, 64-bit logarithms, k rounds, bisections.  One request of four beams 9.7 us, 13 x 5 fp32 15.6.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "beam_step.h"
#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32, kVectors = 16, kList = 256, kPlaces = 6, kWaitLimit = 1 << 22;      // kVectors: pieces of 16 bytes of a thread; kPlaces: CTAs of an SM, as their parts leave room
constexpr int kPart = kThreads * kVectors;                                            // pieces of a part at most
constexpr int kMostParts = 64;                                                         // two of a lane in the second kernel
static_assert(kMostParts * 4 * (kPart - 1) > beam::kMaxVocab && kWarps >= 4 && 4 * 32 >= beam::kMaxFound, "");
constexpr int kLeastPart = 512;                                                       // pieces of a part at least, where the row has them: one request of four beams 9.7 us, of parts of twice that 9.85
constexpr float kLog2e = 1.4426950408889634f;

struct PartHead {
  float top;      // the part's largest logit
  int n;          // candidates
  double sum;     // of exp(x - top)
};
struct Geometry {
  int parts;
  size_t entries;      // byte offset of the candidates behind the heads
  size_t bytes;
};
Geometry geometry(const b200_beam_select_args& a) {
  const long long rows = static_cast<long long>(a.S) * a.beams;
  const int per = a.logits_f32 ? 4 : 8, pieces = (a.V + per - 1) / per;
  // as many parts as fill the SMs' places, of no less than kLeastPart pieces, and as many as hold the row
  const long long wanted = std::min<long long>(kPlaces * sm_count() / std::max<long long>(1, rows), pieces / kLeastPart);
  Geometry g;
  g.parts = static_cast<int>(std::min<long long>(kMostParts, std::max<long long>((pieces + kPart - 1) / kPart, std::max<long long>(1, wanted))));
  g.entries = static_cast<size_t>(rows) * g.parts * sizeof(PartHead);
  g.bytes = g.entries + static_cast<size_t>(rows) * g.parts * a.k * sizeof(uint2);
  return g;
}

// a float's order as an integer's; -0 and 0 are one value
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
// larger for a larger value, and of equal ones for a lower token
__device__ __forceinline__ unsigned long long key_of(float x, int token) { return static_cast<unsigned long long>(order_of(x)) << 32 | static_cast<uint32_t>(~token); }
__device__ __forceinline__ float key_value(unsigned long long k) { return value_of(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int key_token(unsigned long long k) { return static_cast<int>(~static_cast<uint32_t>(k)); }

// Value i of a piece, whose words are given
template <bool kF32>
__device__ __forceinline__ float value_in(const uint32_t* w, int i) {
  if (kF32) return __uint_as_float(w[i]);
  return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
}

// A row's piece, the values of 16 bytes, by the widest loads that the row's beginning allows (which values meet in a sum goes by their tokens alone: equal rows have equal sums wherever they lie).
// What is behind the row's end is -inf.
template <bool kF32, int kAlign>
__device__ __forceinline__ void load_piece(const uint8_t* row, int V, int piece, uint32_t* w) {
  constexpr int kPer = kF32 ? 4 : 8, kSize = kF32 ? 4 : 2;
  const uint8_t* at = row + static_cast<size_t>(piece) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = kF32 ? 0xff800000u : 0xff80ff80u;
  if ((piece + 1) * kPer <= V) {
    if constexpr (kAlign == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(at), v = *reinterpret_cast<const uint2*>(at + 8);
      w[0] = u.x; w[1] = u.y; w[2] = v.x; w[3] = v.y;
    } else if constexpr (kAlign == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(at)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint16_t*>(at)[2 * i] | static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at)[2 * i + 1]) << 16;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer - 1; ++i) {      // (not all of them)
      if (piece * kPer + i >= V) continue;
      if constexpr (kF32) w[i] = reinterpret_cast<const uint32_t*>(at)[i];
      else w[i / 2] = __byte_perm(w[i / 2], *reinterpret_cast<const uint16_t*>(at + i * kSize), i & 1 ? 0x5410 : 0x3254);
    }
  }
}
__device__ __forceinline__ __nv_bfloat162 bf16x2_of(uint32_t w) {
  __nv_bfloat162 p;
  *reinterpret_cast<uint32_t*>(&p) = w;
  return p;
}
template <bool kF32>
__device__ __forceinline__ uint32_t largest_in(const uint4& u) {      // as a word: of bf16 one for each half
  if (kF32) return __float_as_uint(fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w))));
  const __nv_bfloat162 p[4] = {bf16x2_of(u.x), bf16x2_of(u.y), bf16x2_of(u.z), bf16x2_of(u.w)};
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// the bits of those values of a word that are at least this one, which is a value of the type
template <bool kF32>
__device__ __forceinline__ uint32_t those_at_least(uint32_t w, float least) {
  if (kF32) return __uint_as_float(w) >= least ? ~0u : 0u;
  return __hge2_mask(bf16x2_of(w), __float2bfloat162_rn(least));
}
// NaN becomes -inf
template <bool kF32>
__device__ __forceinline__ void without_nan(uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kF32) w[i] = __float_as_uint(fmaxf(__uint_as_float(w[i]), -INFINITY));
    else {
      __nv_bfloat162 p;
      *reinterpret_cast<uint32_t*>(&p) = w[i];
      p = __hmax2(p, __halves2bfloat162(__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80)));
      w[i] = *reinterpret_cast<uint32_t*>(&p);
    }
  }
}

// A row's pieces in parts: `more` of them have one more than `each`
struct Cut {
  int parts, each, more;
};

template <bool kF32>
__global__ void __launch_bounds__(kThreads, kPlaces)
beam_parts_kernel(const __grid_constant__ b200_beam_select_args a, const Cut cut, size_t entries, int* error) {
  constexpr int kPer = kF32 ? 4 : 8;
  constexpr uint32_t kNone = kF32 ? 0xff800000u : 0xff80ff80u;
  extern __shared__ uint4 here[];      // the part
  __shared__ __align__(8) uint64_t bar_word;
  __shared__ uint32_t mosts[kWarps], bounds[kWarps];
  __shared__ double sums[kWarps];
  __shared__ unsigned long long list[kList], sorted[kList];
  __shared__ int s_n, s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned number = blockIdx.x, row = number / static_cast<unsigned>(cut.parts), part = number - row * cut.parts;      // (64-bit quotients were a third of the kernel's instructions)
  const uint8_t* base = static_cast<const uint8_t*>(a.logits) + static_cast<size_t>(row) * a.ld * (kF32 ? 4 : 2);
  const int v0 = part * cut.each + min(static_cast<int>(part), cut.more), count = cut.each + (static_cast<int>(part) < cut.more);
  const int align = static_cast<int>(reinterpret_cast<uintptr_t>(base) & 15);
  const int whole = align ? 0 : min(count, a.V / kPer - v0);      // pieces that a bulk copy brings: those of a row on 16 bytes that its end does not cut
  const uint32_t bar = smem_u32(&bar_word);
  if (tid == 0) {
    mbar_init(bar, 1);
    fence_mbar_init();
    s_n = 0;
  }
  griddep_enter();
  bool ok = true;
  if (tid == 0 && whole > 0) {
    mbar_arrive_expect_tx(bar, static_cast<uint32_t>(whole) * 16);
    bulk_load_1d(smem_u32(here), base + static_cast<size_t>(v0) * 16, static_cast<uint32_t>(whole) * 16, bar);
  }
  // the others go the same way, and behind the last are pieces of nothing: a thread's own, which it alone reads
  const int slots = (count + kThreads - 1) / kThreads;
  for (int i = max(0, whole) / kThreads * kThreads + tid; i < slots * kThreads; i += kThreads) {
    if (i < whole) continue;
    uint32_t w[4] = {kNone, kNone, kNone, kNone};
    if (i < count) {
      if (align % 8 == 0) load_piece<kF32, 8>(base, a.V, v0 + i, w);
      else if (align % 4 == 0) load_piece<kF32, 4>(base, a.V, v0 + i, w);
      else load_piece<kF32, kF32 ? 4 : 2>(base, a.V, v0 + i, w);
    }
    here[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __syncthreads();      // (the barrier's first phase is known to all)
  if (whole > 0) ok = mbar_wait_limited(bar, 0, kWaitLimit);
  // ---- the largest of every piece, two of bf16, and of all
  uint32_t tops[kVectors];
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    tops[v] = kNone;
    if (v < slots) tops[v] = largest_in<kF32>(here[v * kThreads + tid]);
  }
  float mine = -INFINITY;
#pragma unroll
  for (int v = 0; v < kVectors; v += 4) {
    auto at = [&](int i) { return tops[min(i, kVectors - 1)]; };
    const uint32_t m = largest_in<kF32>(make_uint4(at(v), at(v + 1), at(v + 2), at(v + 3)));
    mine = fmaxf(mine, kF32 ? __uint_as_float(m) : fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)));
  }
  // ---- the warp's largest, and the r-th largest of its lanes' maxima (equal ones, which a lane each has, are counted once a round)
  const int r = (a.k + 3) / 4;
  const uint32_t order = order_of(mine), most = __reduce_max_sync(0xffffffffu, order);
  uint32_t rth = most;
  {
    int below = __popc(__ballot_sync(0xffffffffu, order == most));
    while (below < r) {
      rth = __reduce_max_sync(0xffffffffu, order < rth ? order : 0u);
      below += __popc(__ballot_sync(0xffffffffu, order == rth));
    }
  }
  if (lane == 0) {
    mosts[warp] = most;
    bounds[warp] = rth;
  }
  if (!__syncthreads_and(ok)) {      // (a thread that saw the copy come goes on past it: it has come)
    if (tid == 0) *reinterpret_cast<volatile int*>(error) = 1;
    if (whole > 0) mbar_wait_limited(bar, 0, kWaitLimit);
    return;
  }
  const float top = value_of(__reduce_max_sync(0xffffffffu, mosts[lane & (kWarps - 1)]));
  PartHead* head = static_cast<PartHead*>(a.workspace) + number;
  if (top == -INFINITY) {      // nothing here is a candidate
    if (tid == 0) *head = {-INFINITY, 0, 0.0};
    return;
  }
  // the fourth largest of the warps' bounds: four warps have r lanes each that reach it
  uint32_t bound = bounds[lane & (kWarps - 1)];
  {
    int place = 0;
#pragma unroll
    for (int o = 1; o < kWarps; ++o) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, bound, o);
      place += other > bound || (other == bound && ((lane ^ o) & (kWarps - 1)) < (lane & (kWarps - 1)));
    }
    bound = __reduce_max_sync(0xffffffffu, place == 3 ? bound : 0u);
  }
  bound = max(bound, order_of(kF32 ? -FLT_MAX : __uint_as_float(0xff7f0000u)));      // the type's lowest value is one, -inf is none
  const float least = value_of(bound);
  // ---- the list, and the sum of the others
  // exp(x - top) = 2^(x L + c) 2^-(top L + c) for any c: the product inside the sum is exact, so with c near -top L each term has one rounding, and what c's own took from all of them comes
  // back in 64 bits at the end.  (Where top is so large that this does not fit, the difference is taken first.)
  const float from = -top * kLog2e;
  const bool far = !(fabsf(top) < 1048576.f);
  // the list: every lane goes through its own pieces that reach the bound, one or two in all, and takes what does out of them
  uint32_t pieces_left = 0;
#pragma unroll
  for (int v = 0; v < kVectors; ++v)
    if (those_at_least<kF32>(tops[v], least)) pieces_left |= 1u << v;
  for (; pieces_left; pieces_left &= pieces_left - 1) {
    const int at = (__ffs(pieces_left) - 1) * kThreads + tid;
    const uint4 u = here[at];
    uint32_t w[4] = {u.x, u.y, u.z, u.w}, found = 0;      // bit j: the value, or the lower one, of word j; bit 16 + j: the upper one
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t is = those_at_least<kF32>(w[j], least);
      found |= is & ((kF32 ? 0x00000001u : 0x00010001u) << j);
      w[j] = (w[j] & ~is) | (kNone & is);
    }
    here[at] = make_uint4(w[0], w[1], w[2], w[3]);
    for (; found; found &= found - 1) {
      const int bit = __ffs(found) - 1, k = kF32 ? bit : 2 * (bit & 15) + (bit >> 4), word = kF32 ? bit : bit & 15, to = atomicAdd(&s_n, 1);
      const uint32_t x = word & 2 ? (word & 1 ? u.w : u.z) : (word & 1 ? u.y : u.x);
      if (to < kList) list[to] = key_of(kF32 ? __uint_as_float(x) : __uint_as_float(bit & 16 ? x & 0xffff0000u : x << 16), (v0 + at) * kPer + k);
    }
  }
  __syncwarp();      // else the lanes of each way go through the sum by themselves: 3.6 times the exponentials
  float rest;
  for (int again = 0;; ++again) {
    float part_of[4] = {0.f, 0.f, 0.f, 0.f};
    if (!far) {
      const uint64_t scale2 = pair_of(kLog2e, kLog2e), from2 = pair_of(from, from);
      uint64_t two[2] = {0, 0};
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        if (v >= slots) break;
        const uint4 u = here[v * kThreads + tid];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < kPer; k += 2) {
          const float2 x = floats_of(fma_pair(pair_of(value_in<kF32>(w, k), value_in<kF32>(w, k + 1)), scale2, from2));
          two[k / 2 & 1] = add_pair(two[k / 2 & 1], pair_of(exp2_ftz(x.x), exp2_ftz(x.y)));
        }
      }
      const float2 t0 = floats_of(two[0]), t1 = floats_of(two[1]);
      part_of[0] = t0.x; part_of[1] = t0.y; part_of[2] = t1.x; part_of[3] = t1.y;
    } else {
#pragma unroll 1
      for (int v = 0; v < slots; ++v) {
        const uint4 u = here[v * kThreads + tid];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < kPer; ++k) part_of[k & 3] += exp2_ftz((value_in<kF32>(w, k) - top) * kLog2e);
      }
    }
    rest = (part_of[0] + part_of[1]) + (part_of[2] + part_of[3]);
    if (__all_sync(0xffffffffu, rest == rest) || again) break;
    // NaN among the logits: once more without them
#pragma unroll 1
    for (int v = 0; v < slots; ++v) {
      const uint4 u = here[v * kThreads + tid];
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
      without_nan<kF32>(w);
      here[v * kThreads + tid] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncthreads();
  int n = s_n;
  const bool slow = n > kList;
  if (slow) {
    // ---- more than the list holds: the k-th value, bit by bit, over the logits as they lie in L2
    auto each = [&](auto what) {
#pragma unroll 1
      for (int piece = v0 + tid; piece < v0 + count; piece += kThreads) {
        uint32_t w[4];
        load_piece<kF32, kF32 ? 4 : 2>(base, a.V, piece, w);
        without_nan<kF32>(w);
#pragma unroll
        for (int i = 0; i < kPer; ++i) what(value_in<kF32>(w, i), piece * kPer + i);
      }
    };
    auto count_all = [&](auto is) {
      int count = 0;
      each([&](float f, int token) { count += is(order_of(f), token); });
      __syncthreads();
      if (tid == 0) s_count = 0;
      __syncthreads();
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0) atomicAdd(&s_count, count);
      __syncthreads();
      return s_count;
    };
    uint32_t kth = 0;
    for (int bit = 31; bit >= 0; --bit)
      if (count_all([&](uint32_t o, int) { return o >= (kth | 1u << bit); }) >= a.k) kth |= 1u << bit;
    // of the values equal to it those of the lowest tokens: up to the largest `end` that fewer than `wanted` of them lie in front of
    const int wanted = a.k - count_all([&](uint32_t o, int) { return o > kth; });
    int end = 0;
    for (int bit = 18; bit >= 0; --bit)
      if (count_all([&](uint32_t o, int token) { return o == kth && token < (end | 1 << bit); }) < wanted) end |= 1 << bit;
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
    rest = 0.f;
    each([&](float f, int token) {
      const uint32_t o = order_of(f);
      if (o > kth || (o == kth && token <= end)) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kList) list[at] = key_of(f, token);
      } else if (f == top) rest += 1.f;
      else rest += exp2_ftz((f - top) * kLog2e);
    });
    __syncthreads();
    n = min(s_n, kList);
  }
  // ---- places in the list, eight threads a value, and the sum
  double sum = rest;      // (of the slow way: relative to top itself)
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  uint2* out = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.workspace) + entries) + static_cast<size_t>(number) * a.k;
  for (int i0 = 0; i0 < n; i0 += kThreads / 8) {
    const int i = i0 + (tid >> 3);
    const unsigned long long key = list[min(i, n - 1)];
    int place = 0;
    for (int j = tid & 7; j < n; j += 8) place += list[j] > key;
#pragma unroll
    for (int o = 4; o; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
    if (i < n && (tid & 7) == 0) sorted[place] = key;
  }
  __syncthreads();
  if (warp == 0) {      // in the values' order, not in the list's
    double all = lane < kWarps ? sums[lane] * (far || slow ? 1.0 : exp2(-(static_cast<double>(top) * kLog2e + from))) : 0.0;
    for (int i = lane; i < n; i += 32) {
      const unsigned long long key = sorted[i];
      const float f = key_value(key);
      all += f == top ? 1.0 : exp(static_cast<double>(f) - top);
      if (i < a.k) out[i] = make_uint2(static_cast<uint32_t>(key), static_cast<uint32_t>(key >> 32));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) *head = {top, min(n, a.k), all};
  }
}

constexpr int kJoinThreads = 256, kStaged = kMostParts * beam::kMaxFound;      // kStaged: candidates of as many beams as there is room for, one at least

__global__ void __launch_bounds__(kJoinThreads)
beam_join_kernel(const __grid_constant__ b200_beam_select_args a, int parts, size_t entries, int at_once) {
  __shared__ unsigned long long best[beam::kMaxBeams][beam::kMaxFound];      // a beam's, in order
  __shared__ double c_of[beam::kMaxBeams][beam::kMaxFound], offset[beam::kMaxBeams];                                 // c = offset + (x - top), top's own 0
  __shared__ float tops[beam::kMaxBeams];
  __shared__ int count[beam::kMaxBeams], found_token[beam::kMaxFound], found_parent[beam::kMaxFound], ends_text[beam::kMaxFound];
  __shared__ float found_score[beam::kMaxFound];
  __shared__ int places[beam::kMaxBeams][beam::kMaxFound], s_ends[beam::kMaxEnds];
  extern __shared__ unsigned long long staged[];
  __shared__ uint8_t counts[beam::kMaxBeams * kMostParts];
  const int s = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = a.beams, k = a.k;
  griddep_enter();
  const PartHead* heads = static_cast<const PartHead*>(a.workspace) + static_cast<size_t>(s) * B * parts;
  const uint2* lists = reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.workspace) + entries) + static_cast<size_t>(s) * B * parts * k;
  for (int i = tid; i < a.num_ends; i += kJoinThreads) s_ends[i] = a.ends[i];
  for (int i = tid; i < B * k; i += kJoinThreads) places[i / k][i % k] = 0;
  auto sums_of_rows = [&] {
    for (int b = warp; b < B; b += kJoinThreads / 32) {      // a lane has a part
      PartHead h[2];
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int p = lane + 32 * i;
        h[i] = p < parts ? heads[b * parts + p] : PartHead{-INFINITY, 0, 0.0};
        h[i].n = min(max(h[i].n, 0), k);      // whatever a part left whose wait ran out
        if (p < parts) counts[b * parts + p] = h[i].n;
        top = fmaxf(top, h[i].top);
      }
      const float score = a.scores[static_cast<size_t>(s) * B + b];
      double sum = 0.0;
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (h[i].top != -INFINITY) sum += h[i].top == top ? h[i].sum : h[i].sum * exp(static_cast<double>(h[i].top) - top);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const int n = __reduce_add_sync(0xffffffffu, h[0].n + h[1].n);
      const bool real = score > -INFINITY;      // NaN is none
      if (lane == 0) {
        offset[b] = real && n ? score - log(sum) : 0.0;
        tops[b] = top;
        count[b] = real ? min(n, k) : 0;
      }
    }
  };
  for (int i = tid; i < beam::kMaxFound; i += kJoinThreads) {
    found_token[i] = found_parent[i] = -1;
    found_score[i] = -INFINITY;
    ends_text[i] = 0;
  }
  // ---- a beam's candidates in order, a warp a beam: the best of the parts' first ones, k times; of as many beams at a time as there is room for
  for (int b0 = 0; b0 < B; b0 += at_once) {
    const int some = min(at_once, B - b0);
    if (b0) __syncthreads();
    for (int e = tid; e < some * parts * k; e += kJoinThreads) {
      const uint2 x = lists[static_cast<size_t>(b0) * parts * k + e];
      staged[e] = static_cast<unsigned long long>(x.y) << 32 | x.x;      // (what lies behind a part's last is not looked at)
    }
    if (!b0) sums_of_rows();      // under the lists' loads
    __syncthreads();
    for (int b = b0 + warp; b < b0 + some; b += kJoinThreads / 32) {
      const unsigned long long* mine = staged + static_cast<size_t>(b - b0) * parts * k;
      int at[2] = {0, 0};
      unsigned long long first[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) first[i] = lane + 32 * i < parts && counts[b * parts + lane + 32 * i] ? mine[(lane + 32 * i) * k] : 0ull;      // (0 is below every value)
      const int n = count[b];
      const double off = offset[b];
      const float top = tops[b];
      for (int i = 0; i < n; ++i) {
        const bool second = first[1] > first[0];
        const unsigned long long key = second ? first[1] : first[0];
        const uint32_t hi = static_cast<uint32_t>(key >> 32), most = __reduce_max_sync(0xffffffffu, hi);
        bool wins = hi == most;
        if (__popc(__ballot_sync(0xffffffffu, wins)) > 1) {      // equal values: the lowest token (they are all different)
          const uint32_t low = __reduce_max_sync(0xffffffffu, wins ? static_cast<uint32_t>(key) : 0u);
          wins = wins && static_cast<uint32_t>(key) == low;
        }
        if (wins) {
          best[b][i] = key;
          const float x = value_of(most);
          c_of[b][i] = off + (x == top ? 0.0 : static_cast<double>(x) - top);
          const int p = lane + 32 * second, next = (second ? ++at[1] : ++at[0]);
          const unsigned long long follows = next < counts[b * parts + p] ? mine[p * k + next] : 0ull;
          if (second) first[1] = follows;
          else first[0] = follows;
        }
      }
    }
  }
  __syncthreads();
  // ---- and a request's: a candidate's place is its own among its beam's, and how many of every other beam's are ahead of it
  for (int e = tid; e < B * k * B; e += kJoinThreads) {
    const int o = e % B, i = e / B % k, b = e / B / k;
    if (i >= count[b] || !(c_of[b][i] > -INFINITY)) continue;
    const double c = c_of[b][i];
    int lo = o == b ? i : 0, hi = o == b ? i : count[o];
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      const double other = c_of[o][mid];
      if (other > c || (other == c && o < b)) lo = mid + 1;
      else hi = mid;
    }
    if (lo) atomicAdd(&places[b][i], lo);
  }
  __syncthreads();
  for (int e = tid; e < B * k; e += kJoinThreads) {
    const int b = e / k, i = e % k;
    if (i >= count[b] || !(c_of[b][i] > -INFINITY) || places[b][i] >= k) continue;
    const int token = key_token(best[b][i]), place = places[b][i];
    found_token[place] = token;
    found_parent[place] = b;
    found_score[place] = static_cast<float>(c_of[b][i]);
    bool ends = false;
    for (int x = 0; x < a.num_ends; ++x) ends = ends || s_ends[x] == token;
    ends_text[place] = ends;
  }
  __syncthreads();
  for (int i = tid; i < k; i += kJoinThreads) {
    const size_t at = static_cast<size_t>(s) * k + i;
    a.found_parents[at] = found_parent[i];
    a.found_tokens[at] = found_token[i];
    a.found_scores[at] = found_score[i];
  }
  if (warp == 1) {      // those that do not end go on, in order
    const bool goes[2] = {found_parent[lane] >= 0 && !ends_text[lane], found_parent[lane + 32] >= 0 && !ends_text[lane + 32]};
    const unsigned first = __ballot_sync(0xffffffffu, goes[0]), rest = __ballot_sync(0xffffffffu, goes[1]);
    const int all = __popc(first) + __popc(rest);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int to = h ? __popc(first) + __popc(rest & ((1u << lane) - 1)) : __popc(first & ((1u << lane) - 1)), i = lane + 32 * h;
      if (!goes[h] || to >= B) continue;
      const size_t at = static_cast<size_t>(s) * B + to;
      a.parents[at] = found_parent[i];
      a.tokens[at] = found_token[i];
      a.new_scores[at] = found_score[i];
    }
    if (lane >= all && lane < B) {
      const size_t at = static_cast<size_t>(s) * B + lane;
      a.parents[at] = a.tokens[at] = -1;
      a.new_scores[at] = -INFINITY;
    }
  }
}

}  // namespace

int64_t beam_select_workspace(const b200_beam_select_args& a) { return static_cast<int64_t>(geometry(a).bytes); }

int beam_select(const b200_beam_select_args& a, int* error, cudaStream_t st) {
  const Geometry g = geometry(a);
  const int per = a.logits_f32 ? 4 : 8, pieces = (a.V + per - 1) / per;
  const Cut cut = {g.parts, pieces / g.parts, pieces % g.parts};
  const int slots = (cut.each + (cut.more > 0) + kThreads - 1) / kThreads;
  auto kernel = a.logits_f32 ? beam_parts_kernel<true> : beam_parts_kernel<false>;
  static std::atomic<unsigned long long> parts_done[2]{};
  if (!ensure_dynamic_smem(kernel, kPart * 16, &parts_done[!!a.logits_f32])) return -3;
  launch_pdl(kernel, dim3(static_cast<unsigned>(a.S) * a.beams * g.parts), dim3(kThreads), static_cast<size_t>(slots) * kThreads * 16, st, a, cut, g.entries, error);
  if (cudaGetLastError() != cudaSuccess) return -2;
  static std::atomic<unsigned long long> attr_done{0};
  if (!ensure_dynamic_smem(beam_join_kernel, kStaged * 8, &attr_done)) return -3;
  const int at_once = std::min(a.beams, kStaged / (g.parts * a.k));
  launch_pdl(beam_join_kernel, dim3(a.S), dim3(kJoinThreads), static_cast<size_t>(at_once) * g.parts * a.k * 8, st, a, g.parts, g.entries, at_once);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
