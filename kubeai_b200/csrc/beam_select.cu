// The best candidates over a request's beams and the vocabulary.
//
//   c(b, v) = score_b + x_bv - m_b - log sum_w exp(x_bw - m_b)        m_b = max_w x_bw
//
// A row's best candidates by c are its best by x, which needs no rounding, so one pass over the logits takes them by x, together with the sum; c, which decides between beams, is
// made in 64 bits for a few hundred candidates.
// First kernel: a row is cut into parts of at most 16384 bf16 (8192 fp32) logits, a CTA each, whose values stay in registers.  A lower bound of the k-th largest value that few values besides the
// k best reach: of every warp the r-th largest of its lanes' maxima (r = k / 4), and of those the fourth largest, as four warps have r lanes each that reach it.  What does goes to a list,
// where each one's place is the number of better ones.  Where more reach it than the list holds (rows of equal values), the k-th value and the last token that still belongs are found bit by bit over all values.
// The sum's large terms, those of the list, are taken in 64 bits, the others as 2^t in 32, t in two products: what an fp32 sum loses would decide between beams whose candidates lie close
// together.
// Second kernel, a CTA a request: a candidate's place among those of all parts, then of all beams, is its place in its own list and, by bisection, in every other.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "beam_step.h"
#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kVectors = 8, kList = 256, kPlaces = 4, kAtOnce = 4;      // kVectors: pieces of 16 bytes of a thread; kPlaces: CTAs of an SM; kAtOnce: threads' values on their way to the list
constexpr int kPart = kThreads * kVectors;                                            // pieces of a part at most
constexpr int kMostParts = 64;                                                         // two of a lane in the second kernel
static_assert(kMostParts * 4 * (kPart - 1) > beam::kMaxVocab && kWarps >= 4 && 4 * 32 >= beam::kMaxFound, "");
constexpr int kLeastPart = 1024;                                                       // pieces of a part at least, where the row has them
constexpr float kLog2eHi = 1.4426950216293335f, kLog2eLo = 1.9259629911e-8f;           // log2(e) as a sum

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
__device__ __forceinline__ void load_piece(const uint8_t* row, int V, int piece, bool there, uint32_t* w) {
  constexpr int kPer = kF32 ? 4 : 8, kSize = kF32 ? 4 : 2;
  const uint8_t* at = row + static_cast<size_t>(piece) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = kF32 ? 0xff800000u : 0xff80ff80u;
  if (!there) return;
  if ((piece + 1) * kPer <= V) {
    if constexpr (kAlign == 16) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(at));
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (kAlign == 8) {
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
    for (int i = 0; i < kPer; ++i) {
      if (piece * kPer + i >= V) continue;
      if constexpr (kF32) w[i] = reinterpret_cast<const uint32_t*>(at)[i];
      else w[i / 2] = __byte_perm(w[i / 2], *reinterpret_cast<const uint16_t*>(at + i * kSize), i & 1 ? 0x5410 : 0x3254);
    }
  }
}
template <bool kF32>
__device__ __forceinline__ float largest_in(const uint32_t* w) {
  if (kF32) return fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])), fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
  __nv_bfloat162 p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(&p[i]) = w[i];
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
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

template <bool kF32>
__global__ void __launch_bounds__(kThreads, kPlaces)
beam_parts_kernel(const __grid_constant__ b200_beam_select_args a, int parts, size_t entries) {
  constexpr int kPer = kF32 ? 4 : 8;
  __shared__ uint32_t mosts[kWarps], bounds[kWarps];
  __shared__ double sums[kWarps];
  __shared__ unsigned long long list[kList];
  __shared__ double terms[kList];
  __shared__ int s_n, s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  griddep_enter();
  const uint8_t* base = static_cast<const uint8_t*>(a.logits) + static_cast<size_t>(row) * a.ld * (kF32 ? 4 : 2);
  const int pieces = (a.V + kPer - 1) / kPer;
  const int v0 = static_cast<int>(static_cast<long long>(pieces) * part / parts), v1 = static_cast<int>(static_cast<long long>(pieces) * (part + 1) / parts);

  uint32_t x[kVectors][4];
  auto load = [&](auto align) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v) load_piece<kF32, decltype(align)::value>(base, a.V, v0 + v * kThreads + tid, v0 + v * kThreads + tid < v1, x[v]);
  };
  const int align = static_cast<int>(reinterpret_cast<uintptr_t>(base) & 15);
  if (align == 0) load(std::integral_constant<int, 16>());
  else if (align == 8) load(std::integral_constant<int, 8>());
  else if (align % 4 == 0) load(std::integral_constant<int, 4>());
  else load(std::integral_constant<int, 2>());
  float mine = -INFINITY;
#pragma unroll
  for (int v = 0; v < kVectors; ++v) mine = fmaxf(mine, largest_in<kF32>(x[v]));
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
  if (tid == 0) s_n = 0;
  __syncthreads();
  uint32_t all = 0, bound = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all = max(all, mosts[w]);
  const float top = value_of(all);
  PartHead* head = static_cast<PartHead*>(a.workspace) + row * parts + part;
  if (top == -INFINITY) {      // nothing here is a candidate
    if (tid == 0) *head = {-INFINITY, 0, 0.0};
    return;
  }
  {      // the fourth largest of the warps' bounds
    const uint32_t mine4 = bounds[lane % kWarps];
    int place = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) place += bounds[w] > mine4 || (bounds[w] == mine4 && w < lane % kWarps);
    bound = __reduce_max_sync(0xffffffffu, place == 3 ? mine4 : 0u);
  }
  if (bound <= order_of(-INFINITY)) bound = order_of(-INFINITY) + 1;      // the smallest value that is one
  float least = value_of(bound);
  // ---- the sum of those below it, by every thread that has no others
  const uint64_t less = pair_of(-top, -top), hi = pair_of(kLog2eHi, kLog2eHi), lo = pair_of(kLog2eLo, kLog2eLo);
  float rest = 0.f;
  const unsigned some = __ballot_sync(0xffffffffu, mine >= least);
  if (mine < least) {
#pragma unroll 1
    for (int again = 0; again < 2; ++again) {
      uint64_t sum2[2] = {0, 0};
#pragma unroll
      for (int v = 0; v < kVectors; ++v)
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
          const uint64_t d = add_pair(pair_of(value_in<kF32>(x[v], i), value_in<kF32>(x[v], i + 1)), less);
          const float2 t = floats_of(fma_pair(d, hi, mul_pair(d, lo)));
          sum2[v & 1] = add_pair(sum2[v & 1], pair_of(exp2_ftz(t.x), exp2_ftz(t.y)));
        }
      const float2 p = floats_of(sum2[0]), q = floats_of(sum2[1]);
      rest = (p.x + p.y) + (q.x + q.y);
      if (rest == rest) break;
#pragma unroll
      for (int v = 0; v < kVectors; ++v) without_nan<kF32>(x[v]);      // NaN among the logits: once more without them
    }
  }
  // ---- the few threads that have something for the list, one behind the other by their warp: a lane has a word of theirs, from where it lies in L2
  float apart = 0.f;
  for (unsigned left = some; left;) {
    uint32_t word[kAtOnce];
    int token[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int piece = v0 + (lane >> 2) * kThreads + warp * 32 + (left ? __ffs(left) - 1 : 0);
      token[k] = left && piece < v1 ? piece * kPer + (lane & 3) * (kF32 ? 1 : 2) : a.V;
      left &= left - 1;
      word[k] = 0;
      if (token[k] >= a.V) continue;
      if constexpr (kF32) word[k] = reinterpret_cast<const uint32_t*>(base)[token[k]];
      else word[k] = reinterpret_cast<const uint16_t*>(base)[token[k]] | static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(base)[min(token[k] + 1, a.V - 1)]) << 16;
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
#pragma unroll
      for (int i = 0; i < (kF32 ? 1 : 2); ++i) {
        const float f = kF32 ? __uint_as_float(word[k]) : __uint_as_float(i ? word[k] & 0xffff0000u : word[k] << 16), d = f - top;
        if (token[k] + i >= a.V) continue;
        if (f >= least) {
          const int at = atomicAdd(&s_n, 1);
          if (at < kList) list[at] = key_of(f, token[k] + i);
        } else if (f == f) apart += exp2_ftz(fmaf(d, kLog2eHi, d * kLog2eLo));
      }
  }
  rest += apart;
  __syncthreads();
  int n = s_n;
  if (n > kList) {
    // ---- more than the list holds: the k-th value, bit by bit, over the logits as they lie in L2
    auto each = [&](auto what) {
#pragma unroll 1
      for (int piece = v0 + tid; piece < v1; piece += kThreads) {
        uint32_t w[4];
        load_piece<kF32, kF32 ? 4 : 2>(base, a.V, piece, true, w);
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
      else rest += exp2_ftz(fmaf(f - top, kLog2eHi, (f - top) * kLog2eLo));
    });
    __syncthreads();
    n = min(s_n, kList);
  }
  // ---- places in the list, and the sum
  static_assert(kList <= kThreads, "");
  double sum = rest;
  uint2* out = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.workspace) + entries) + (row * parts + part) * a.k;
  for (int i = tid; i < n; i += kThreads) {
    const unsigned long long key = list[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += list[j] > key;
    if (place < a.k) out[place] = make_uint2(static_cast<uint32_t>(key), static_cast<uint32_t>(key >> 32));
    const float f = key_value(key);
    terms[place] = f == top ? 1.0 : exp(static_cast<double>(f) - top);
  }
  __syncthreads();
  if (tid < n) sum += terms[tid];      // in the values' order, not in the list's
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
    for (int w = 0; w < kWarps; ++w) all += sums[w];
    *head = {top, min(n, a.k), all};
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
  extern __shared__ unsigned long long staged[];
  __shared__ uint8_t counts[beam::kMaxBeams * kMostParts];
  const int s = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = a.beams, k = a.k;
  griddep_enter();
  const PartHead* heads = static_cast<const PartHead*>(a.workspace) + static_cast<size_t>(s) * B * parts;
  const uint2* lists = reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.workspace) + entries) + static_cast<size_t>(s) * B * parts * k;
  for (int b = warp; b < B; b += kJoinThreads / 32) {      // a lane has a part
    PartHead h[2];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = lane + 32 * i;
      h[i] = p < parts ? heads[b * parts + p] : PartHead{-INFINITY, 0, 0.0};
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
        const uint32_t low = __reduce_max_sync(0xffffffffu, hi == most ? static_cast<uint32_t>(key) : 0u);      // (tokens are all different)
        if (hi == most && static_cast<uint32_t>(key) == low) {
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
  // ---- and a request's
  for (int e = tid; e < B * k; e += kJoinThreads) {
    const int b = e / k, i = e % k;
    if (i >= count[b]) continue;
    const double c = c_of[b][i];
    if (!(c > -INFINITY)) continue;
    int place = i;
    for (int o = 0; o < B && place < k; ++o) {
      if (o == b) continue;
      int lo = 0, hi = count[o];
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const double other = c_of[o][mid];
        if (other > c || (other == c && o < b)) lo = mid + 1;
        else hi = mid;
      }
      place += lo;
    }
    if (place < k) {
      const int token = key_token(best[b][i]);
      found_token[place] = token;
      found_parent[place] = b;
      found_score[place] = static_cast<float>(c);
      bool ends = false;
      for (int x = 0; x < a.num_ends; ++x) ends = ends || a.ends[x] == token;
      ends_text[place] = ends;
    }
  }
  __syncthreads();
  for (int i = tid; i < k; i += kJoinThreads) {
    const size_t at = static_cast<size_t>(s) * k + i;
    a.found_parents[at] = found_parent[i];
    a.found_tokens[at] = found_token[i];
    a.found_scores[at] = found_score[i];
  }
  for (int i = tid; i < B; i += kJoinThreads) {
    int at = 0;
    for (int left = i; at < k; ++at)
      if (found_parent[at] >= 0 && !ends_text[at] && left-- == 0) break;
    const size_t to = static_cast<size_t>(s) * B + i;
    a.parents[to] = at < k ? found_parent[at] : -1;
    a.tokens[to] = at < k ? found_token[at] : -1;
    a.new_scores[to] = at < k ? found_score[at] : -INFINITY;
  }
}

}  // namespace

int64_t beam_select_workspace(const b200_beam_select_args& a) { return static_cast<int64_t>(geometry(a).bytes); }

int beam_select(const b200_beam_select_args& a, cudaStream_t st) {
  const Geometry g = geometry(a);
  const dim3 grid(static_cast<unsigned>(a.S) * a.beams * g.parts);
  launch_pdl(a.logits_f32 ? beam_parts_kernel<true> : beam_parts_kernel<false>, grid, dim3(kThreads), 0, st, a, g.parts, g.entries);
  if (cudaGetLastError() != cudaSuccess) return -2;
  static std::atomic<unsigned long long> attr_done{0};
  if (!ensure_dynamic_smem(beam_join_kernel, kStaged * 8, &attr_done)) return -3;
  const int at_once = std::min(a.beams, kStaged / (g.parts * a.k));
  launch_pdl(beam_join_kernel, dim3(a.S), dim3(kJoinThreads), static_cast<size_t>(at_once) * g.parts * a.k * 8, st, a, g.parts, g.entries, at_once);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
