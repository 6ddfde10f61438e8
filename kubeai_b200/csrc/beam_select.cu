// The best candidates over a request's beams and the vocabulary.
//
//   c(b, v) = score_b + x_bv - m_b - log sum_w exp(x_bw - m_b)        m_b = max_w x_bw
//
// A row's best candidates by c are its best by x, which needs no rounding, so one pass over the logits takes them by x, together with the sum; c, which decides between beams, is
// made in 64 bits for a few hundred candidates.
// First kernel: a row is cut into parts of at most 32768 bf16 (16384 fp32) logits, a CTA each, whose values stay in registers.  The k-th largest of the threads' maxima is
// a lower bound of the k-th largest value (found bit by bit, 16 counts over the CTA), and few values besides the k best reach it: those go to a list, where each one's place is the number of
// better ones.  Where more reach it than the list holds (rows of equal values), the k-th value and the last token that still belongs are found bit by bit over all values.
// The sum's large terms, those of the list, are taken in 64 bits, the others as 2^t in 32, t in two products: what an fp32 sum loses would decide between beams whose candidates lie close
// together.
// Second kernel, a CTA a request: a candidate's place among those of all parts, then of all beams, is its place in its own list and, by bisection, in every other.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "beam_step.h"
#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kVectors = 8, kList = 512;      // kVectors: pieces of 16 bytes of a thread
constexpr int kPart = kThreads * kVectors;                                            // pieces of a part at most
constexpr int kMostParts = 32;                                                         // a lane each in the second kernel
static_assert(kMostParts * 4 * (kPart - 1) > beam::kMaxVocab, "");
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
  // as many parts as fill the SMs twice, of no less than kLeastPart pieces, and as many as hold the row
  const long long wanted = std::min<long long>(2 * sm_count() / std::max<long long>(1, rows), pieces / kLeastPart);
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

// A row's piece: the values of 16 bytes, by the widest loads that the row's beginning allows, so that which values meet in a sum goes by their tokens alone and equal rows have equal
// sums wherever they lie.  What is behind the row's end is -inf.
template <bool kF32>
__device__ __forceinline__ void load_piece(const uint8_t* row, int V, int piece, bool there, uint32_t* w) {
  constexpr int kPer = kF32 ? 4 : 8, kSize = kF32 ? 4 : 2;
  const uint8_t* at = row + static_cast<size_t>(piece) * 16;
  const int align = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = kF32 ? 0xff800000u : 0xff80ff80u;
  if (!there) return;
  if ((piece + 1) * kPer <= V && align % 4 == 0) {
    if (align == 0) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(at));
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if (align == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(at), v = *reinterpret_cast<const uint2*>(at + 8);
      w[0] = u.x; w[1] = u.y; w[2] = v.x; w[3] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(at)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (piece * kPer + i >= V) continue;
      if (kF32) w[i & 3] = reinterpret_cast<const uint32_t*>(at)[i];
      else w[i / 2] = __byte_perm(w[i / 2], *reinterpret_cast<const uint16_t*>(at + i * kSize), i & 1 ? 0x5410 : 0x3254);
    }
  }
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
__global__ void __launch_bounds__(kThreads, 2)
beam_parts_kernel(const __grid_constant__ b200_beam_select_args a, int parts, size_t entries) {
  constexpr int kPer = kF32 ? 4 : 8;
  __shared__ float maxima[kWarps];
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
#pragma unroll
  for (int v = 0; v < kVectors; ++v) load_piece<kF32>(base, a.V, v0 + v * kThreads + tid, v0 + v * kThreads + tid < v1, x[v]);
  float mine = -INFINITY;
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    without_nan<kF32>(x[v]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine = fmaxf(mine, value_in<kF32>(x[v], i));
  }
  float top = mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) maxima[warp] = top;
  if (tid == 0) s_n = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, maxima[w]);
  PartHead* head = static_cast<PartHead*>(a.workspace) + row * parts + part;
  if (top == -INFINITY) {      // nothing here is a candidate
    if (tid == 0) *head = {-INFINITY, 0, 0.0};
    return;
  }
  // ---- the k-th largest maximum, its upper 16 bits
  const uint32_t order = order_of(mine);
  uint32_t bound = 0;
  for (int bit = 31; bit >= 16; --bit)
    if (__syncthreads_count(order >= (bound | 1u << bit)) >= a.k) bound |= 1u << bit;
  if (bound <= order_of(-INFINITY)) bound = order_of(-INFINITY) + 1;      // the smallest value that is one
  float least = value_of(bound);
  // ---- the list, and the sum of the others
  float rest = 0.f;
#pragma unroll
  for (int v = 0; v < kVectors; ++v)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float f = value_in<kF32>(x[v], i), d = f - top;
      if (f >= least) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kList) list[at] = key_of(f, (v0 + v * kThreads + tid) * kPer + i);
      } else rest += exp2_ftz(fmaf(d, kLog2eHi, d * kLog2eLo));
    }
  __syncthreads();
  int n = s_n;
  if (n > kList) {
    // ---- more than the list holds: the k-th value, bit by bit, over the logits as they lie in L2
    auto each = [&](auto what) {
#pragma unroll 1
      for (int piece = v0 + tid; piece < v1; piece += kThreads) {
        uint32_t w[4];
        load_piece<kF32>(base, a.V, piece, true, w);
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

constexpr int kJoinThreads = 256, kStaged = kMostParts * beam::kMaxFound;

__global__ void __launch_bounds__(kJoinThreads)
beam_join_kernel(const __grid_constant__ b200_beam_select_args a, int parts, size_t entries) {
  __shared__ unsigned long long best[beam::kMaxBeams][beam::kMaxFound];      // a beam's, in order
  __shared__ double offset[beam::kMaxBeams];                                 // c = offset + (x - top), top's own 0
  __shared__ float tops[beam::kMaxBeams];
  __shared__ int count[beam::kMaxBeams], found_token[beam::kMaxFound], found_parent[beam::kMaxFound], ends_text[beam::kMaxFound];
  __shared__ float found_score[beam::kMaxFound];
  __shared__ unsigned long long staged[kStaged];
  __shared__ uint8_t counts[beam::kMaxBeams * kMostParts];
  const int s = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = a.beams, k = a.k;
  griddep_enter();
  const PartHead* heads = static_cast<const PartHead*>(a.workspace) + static_cast<size_t>(s) * B * parts;
  const uint2* lists = reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.workspace) + entries) + static_cast<size_t>(s) * B * parts * k;
  for (int b = warp; b < B; b += kJoinThreads / 32) {      // a lane has a part
    const PartHead h = lane < parts ? heads[b * parts + lane] : PartHead{-INFINITY, 0, 0.0};
    if (lane < parts) counts[b * parts + lane] = h.n;
    const float score = a.scores[static_cast<size_t>(s) * B + b];
    float top = h.top;
    double sum = 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (h.top != -INFINITY) sum = h.top == top ? h.sum : h.sum * exp(static_cast<double>(h.top) - top);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int n = __reduce_add_sync(0xffffffffu, h.n);
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
  __syncthreads();
  // ---- a row's candidates in order, of as many beams at a time as there is room for
  const int at_once = max(1, kStaged / (parts * k));
  for (int b0 = 0; b0 < B; b0 += at_once) {
    const int some = min(at_once, B - b0) * parts;
    for (int e = tid; e < some * k; e += kJoinThreads) {
      const uint2 x = lists[static_cast<size_t>(b0) * parts * k + e];
      staged[e] = e % k < counts[b0 * parts + e / k] ? static_cast<unsigned long long>(x.y) << 32 | x.x : 0ull;      // (0 is below every value)
    }
    __syncthreads();
    for (int e = tid; e < some * k; e += kJoinThreads) {
      const unsigned long long key = staged[e];
      const int list = e / k, b = list / parts;
      if (!key || !count[b0 + b]) continue;
      int place = e % k;
      for (int p = b * parts; p < (b + 1) * parts && place < k; ++p) {
        if (p == list) continue;
        int lo = 0, hi = k;      // how many of its are larger
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (staged[p * k + mid] > key) lo = mid + 1;
          else hi = mid;
        }
        place += lo;
      }
      if (place < k) best[b0 + b][place] = key;
    }
    __syncthreads();
  }
  // ---- and a request's
  auto c_of = [&](int b, int i) {
    const float x = key_value(best[b][i]);
    return offset[b] + (x == tops[b] ? 0.0 : static_cast<double>(x) - tops[b]);
  };
  for (int e = tid; e < B * k; e += kJoinThreads) {
    const int b = e / k, i = e % k;
    if (i >= count[b]) continue;
    const double c = c_of(b, i);
    if (!(c > -INFINITY)) continue;
    int place = i;
    for (int o = 0; o < B && place < k; ++o) {
      if (o == b) continue;
      int lo = 0, hi = count[o];
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const double other = c_of(o, mid);
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
  launch_pdl(beam_join_kernel, dim3(a.S), dim3(kJoinThreads), 0, st, a, g.parts, g.entries);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace b200
