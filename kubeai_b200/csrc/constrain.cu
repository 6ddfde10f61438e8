// Penalties, biases and grammar masks on logits, and the greedy choice, in one pass over the rows.
//
//   y = x;  said anywhere: y = y > 0 ? y / rho : y rho;  y -= phi c;  y -= pi where c > 0;  y += bias;  not allowed: -inf;  id = argmax y
//
// A vocabulary's rows are long and what is said about single tokens is short.  So a cluster of CTAs shares a row, each with a slice of the vocabulary, and
// a CTA marks the tokens of its slice that the request's lists name with a bit each.  The bits' running count gives every such token a slot, where its count,
// its bias and its number lie: as much shared memory as there is to say, whatever the vocabulary.  More tokens than slots: the slice is worked on in pieces
// that have no more.  All of this is done once for the rows of a request that the cluster takes, while the first rows are on their way: a row's part of the
// slice comes as one bulk copy, the next row's behind it, so that neither registers nor a thread's order of loads decide what is in flight.
// A row is then two passes side by side: its vectors from shared memory, of which eight tokens cost a maximum of pairs, marked tokens left out; and the slots,
// a thread each, which alone need the formula.  A row's drafts are counted in ahead of it and out behind it.
// The slices' best pairs (value, token) meet through distributed shared memory.  Ties go to the lowest token: every comparison prefers it.
// Every wait for a copy has a limit; a CTA that gives up sets an error mark.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "tree_step.h"
#include "umma2.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256, kMostCtas = 16, kRows = 256, kAhead = 8, kSlots = 2048, kList = 4096, kPlaces = 3;      // kPlaces: CTAs of an SM
constexpr int kSliceBytes = 32 << 10, kWaitLimit = 1 << 22;
constexpr int kSaid = 0x8000;      // of a place: not in the prompt
constexpr unsigned kPrompt = 0x80000000u, kBiased = 0x40000000u;      // of a count: said in the prompt, which the repetition penalty alone counts; has a bias

__device__ __forceinline__ unsigned long long peer_load(const void* p, unsigned rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_u32(smem_u32(p), rank)) : "memory");
  return v;
}

// A choice's value as a number that is larger for the better one, 0 for none.  Above the token, the lower the larger, the whole choice is one number.
__device__ __forceinline__ unsigned ordered(float y, int id) {
  if (y == 0.f) y = 0.f;      // -0 is no smaller
  const unsigned u = __float_as_uint(y);
  return id < 0 ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sixteen bytes of a row.
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ unsigned word(const uint4& u, int w) { return w == 0 ? u.x : w == 1 ? u.y : w == 2 ? u.z : u.w; }
  static __device__ __forceinline__ float get(const uint4& u, int j) { return __uint_as_float(j & 1 ? word(u, j >> 1) & 0xffff0000u : word(u, j >> 1) << 16); }
  // the largest of the tokens over which keep has ones; NaN only where nothing else is
  static __device__ __forceinline__ float largest(const uint4& u, const uint4& keep) {
    auto pair = [](unsigned v, unsigned k) {
      v = (v & k) | (0xff80ff80u & ~k);
      return *reinterpret_cast<__nv_bfloat162*>(&v);
    };
    const __nv_bfloat162 t = __hmax2(__hmax2(pair(u.x, keep.x), pair(u.y, keep.y)), __hmax2(pair(u.z, keep.z), pair(u.w, keep.w)));
    return fmaxf(__low2float(t), __high2float(t));
  }
  static __device__ __forceinline__ uint4 keep(unsigned ok) {
    auto pair = [&](int j) { return (ok >> j & 1 ? 0xffffu : 0u) | (ok >> (j + 1) & 1 ? 0xffff0000u : 0u); };
    return make_uint4(pair(0), pair(2), pair(4), pair(6));
  }
  static __device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const uint4& u, int j) { return __uint_as_float(j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w); }
  static __device__ __forceinline__ float largest(const uint4& u, const uint4& keep) {
    auto one = [](unsigned v, unsigned k) { return __uint_as_float((v & k) | (0xff800000u & ~k)); };
    return fmaxf(fmaxf(one(u.x, keep.x), one(u.y, keep.y)), fmaxf(one(u.z, keep.z), one(u.w, keep.w)));
  }
  static __device__ __forceinline__ uint4 keep(unsigned ok) { return make_uint4(-(ok & 1), -(ok >> 1 & 1), -(ok >> 2 & 1), -(ok >> 3 & 1)); }
  static __device__ __forceinline__ float value(float v) { return v; }
};

struct None {};
// y[0 .. N) to p, of which only the places `inside` are to be written
template <int N>
__device__ __forceinline__ void store_all(float* p, const float* y, unsigned inside) {
  if (inside == (1u << N) - 1 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
    for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (inside >> j & 1) p[j] = y[j];
  }
}
template <int N>
__device__ __forceinline__ void store_all(__nv_bfloat16* p, const float* y, unsigned inside) {
  if (inside == (1u << N) - 1 && reinterpret_cast<uintptr_t>(p) % (2 * N) == 0) {
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (inside >> j & 1) p[j] = __float2bfloat16_rn(y[j]);
  }
}
__device__ __forceinline__ void store_one(float* p, float y) { *p = y; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float y) { *p = __float2bfloat16_rn(y); }

// Rows that no request owns have no choice (one block).
__device__ void no_choice(const b200_constrain_args& a) {
  bool plain = true;
  for (int i = threadIdx.x; i < a.S; i += kThreads) plain = plain && a.starts[i] >= 0 && a.starts[i] <= a.starts[i + 1] && a.starts[i + 1] <= a.T;
  plain = __syncthreads_and(plain);
  for (int t = threadIdx.x; t < a.T; t += kThreads) {
    bool owned = plain && t >= a.starts[0] && t < a.starts[a.S];
    for (int i = 0; !plain && !owned && i < a.S; ++i) owned = a.starts[i] >= 0 && a.starts[i + 1] <= a.T && t >= a.starts[i] && t < a.starts[i + 1];
    if (!owned) a.ids[t] = -1;
  }
}

// bytes of one of a row's buffers: a slice from its 16-byte boundary on
__host__ __device__ constexpr int buffer_bytes(int slice, int size) { return (slice * size + 15) / 16 * 16 + 16; }

// TIn: the logits; TOut: y kept, or None.  slice: tokens of a CTA, a multiple of 32; buffers: rows on their way, 1 or 2.
template <typename TIn, typename TOut>
__global__ void __launch_bounds__(kThreads, kPlaces)
constrain_kernel(const __grid_constant__ b200_constrain_args a, int slice, int buffers, int* error) {
  constexpr int N = Vec<TIn>::N;
  constexpr unsigned kAll = (1u << N) - 1;
  constexpr bool KEEP = !std::is_same<TOut, None>::value;
  extern __shared__ __align__(16) uint8_t smem[];
  const int slice_words = slice / 32;
  uint8_t* buffer = smem;
  unsigned* known = reinterpret_cast<unsigned*>(smem + buffers * buffer_bytes(slice, sizeof(TIn)));      // [slice_words + 1] the slice's tokens that the lists name
  unsigned* may = known + slice_words + 1;                             // [slice_words + 1] those that the row's mask allows
  int* slot_of = reinterpret_cast<int*>(may + slice_words + 1);        // [slice_words] marked tokens in front of each word
  __shared__ unsigned count[kSlots];               // how often the token was said, with the marks above
  __shared__ int entry[kSlots];                    // the last bias entry, then the bias
  __shared__ uint16_t token[kSlots];               // places in the slice
  __shared__ uint16_t list[kList];                 // the history's tokens that are the slice's, by their places, with kSaid
  __shared__ unsigned long long best_of[kRows];
  __shared__ uint4 keep_of[1 << N];                // Vec<TIn>::keep of every set of a vector's tokens
  __shared__ int sums[kThreads / 32], s_end, listed;
  __shared__ uint64_t bar[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = static_cast<int>(cluster_ctarank()), ctas = gridDim.x;
  const int lo = rank * slice, size = max(0, min(slice, a.V - lo));
  const int s = blockIdx.z, group = blockIdx.y, groups = gridDim.y;
  if (tid == 0) {
    for (int b = 0; b < 2; ++b) mbar_init(smem_u32(bar + b), 1);
    fence_mbar_init();
    listed = 0;
  }
  // ids may be read by a kernel behind this one ahead of its dependency wait: none is let in before the end
  griddep_wait();
  if (s == a.S) {
    if (!group && !rank) no_choice(a);
    return;
  }
  // (everything that is looked up by the request alone is on its way at once)
  int row0 = s, rows = 1, h0 = 0, h1 = 0, prompt = 0, b0 = 0, b1 = 0;
  float rho = 1.f, pi = 0.f, phi = 0.f;
  if (a.starts) row0 = a.starts[s], rows = a.starts[s + 1];
  if (a.penalties) rho = a.penalties[3 * s], pi = a.penalties[3 * s + 1], phi = a.penalties[3 * s + 2];
  if (a.history) {
    h0 = a.hist_starts[s], h1 = a.hist_starts[s + 1];
    if (a.prompt_lens) prompt = a.prompt_lens[s];
  }
  if (a.bias_starts) b0 = a.bias_starts[s], b1 = a.bias_starts[s + 1];
  if (a.starts) rows = row0 >= 0 && rows >= row0 && rows <= a.T ? rows - row0 : 0;
  h0 = max(h0, 0), h1 = min(h1, a.history_len);
  b0 = max(b0, 0), b1 = min(b1, a.bias_len);
  if (group >= rows) return;      // (the whole cluster)
  const int my_rows = (rows - group + groups - 1) / groups;
  __syncthreads();

  // ---- a row's part of the piece [from, from + tokens) of the slice: its whole 16 bytes by a copy, the others by threads (warp 0)
  int from = 0, tokens = size, issued = 0;      // copies so far
  auto skew_of = [&](const TIn* p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(TIn) % N); };      // tokens between a 16-byte boundary and p
  auto row_at = [&](int d) { return static_cast<const TIn*>(a.logits) + static_cast<size_t>(row0 + group + d * groups) * a.ld + lo + from; };
  auto fetch = [&](int d) {
    const TIn* p = row_at(d);
    const int skew = skew_of(p), head = min(tokens, (N - skew) % N), whole = (tokens - head) / N, tail = tokens - head - whole * N;
    TIn* dst = reinterpret_cast<TIn*>(buffer + (issued % buffers) * buffer_bytes(slice, sizeof(TIn))) + skew;      // of token 0
    const uint32_t b = smem_u32(bar + issued % buffers);
    if (lane < head) dst[lane] = p[lane];
    if (lane < tail) dst[head + whole * N + lane] = p[head + whole * N + lane];
    if (lane == 0) {
      mbar_arrive_expect_tx(b, whole * 16);
      if (whole) bulk_load_1d(smem_u32(dst + head), p + head, whole * 16, b);
    }
  };
  auto fetch_next = [&](int d) {
    if (warp == 0) fetch(d);
    ++issued;
  };
  for (int d = 0; d < min(buffers, my_rows); ++d) fetch_next(d);

  auto place = [&](int v) { return v >= lo && v < lo + size ? v - lo : -1; };      // in the slice

  // ---- which tokens of the slice the lists name.  The history's are noted down on the way, so that counting them need not look at the others again.  What a
  // thread takes first of the biases and drafts stays in its registers.
  int bias_at = -1, draft_at = -1;
  float bias_value = 0.f;
  if (b0 + tid < b1) bias_at = a.bias_ids[b0 + tid], bias_value = a.bias_values[b0 + tid];
  if (a.drafts && tid < rows) draft_at = a.drafts[row0 + tid];
  int ahead[kAhead];
  auto look = [&](int base) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int i = base + e * kThreads + tid;
      ahead[e] = i < h1 ? a.history[i] : -1;
    }
  };
  look(h0);
  auto mask_word = [&](int d) -> unsigned {      // of the cluster's row d, the one with this thread's draft
    const int i = group + d * groups;
    return !a.drafts || i >= rows ? 0u : !a.masks ? (tid <= i ? ~0u : 0u) : (tid >> 5) < a.words ? static_cast<unsigned>(a.masks[static_cast<size_t>(row0 + i) * a.words + (tid >> 5)]) : 0u;
  };
  auto allow_of = [&](int d) -> const unsigned* {      // its mask's words of the slice
    const int i = group + d * groups;
    if (!a.allow || i >= rows) return nullptr;
    const int m = a.allow_rows ? a.allow_rows[row0 + i] : row0 + i;
    return m >= 0 && m < a.allow_count ? reinterpret_cast<const unsigned*>(a.allow) + static_cast<size_t>(m) * a.ld_allow + lo / 32 : nullptr;
  };
  for (int w = tid; w <= slice_words; w += kThreads) known[w] = 0, may[w] = ~0u;
  for (int d = tid; d < kRows; d += kThreads) best_of[d] = 0;
  for (int d = tid; d < 1 << N; d += kThreads) keep_of[d] = Vec<TIn>::keep(d);
  bias_at = place(bias_at);
  draft_at = place(draft_at);
  __syncthreads();
  auto know = [&](int k) {
    if (k >= 0) atomicOr(known + (k >> 5), 1u << (k & 31));
  };
  auto history = [&](auto f) {      // f(place, said in the prompt)
    for (int base = h0; base < h1; base += kAhead * kThreads) {
#pragma unroll
      for (int e = 0; e < kAhead; ++e) f(place(ahead[e]), base + e * kThreads + tid - h0 < prompt);
      if (base + kAhead * kThreads < h1) look(base + kAhead * kThreads);
    }
  };
  history([&](int k, bool in_prompt) {
    if (k < 0) return;
    const int at = atomicAdd(&listed, 1);
    if (at < kList) list[at] = static_cast<uint16_t>(k | (in_prompt ? 0 : kSaid));
    know(k);
  });
  know(bias_at);
  for (int i = b0 + kThreads + tid; i < b1; i += kThreads) know(place(a.bias_ids[i]));
  know(draft_at);
  if (a.drafts)
    for (int i = kThreads + tid; i < rows; i += kThreads) know(place(a.drafts[row0 + i]));
  __syncthreads();
  // slots: a thread sums some words, one behind the other
  const int per = (slice_words + kThreads - 1) / kThreads, w_begin = min(slice_words, tid * per), w_end = min(slice_words, w_begin + per);
  int before = 0;
  for (int w = w_begin; w < w_end; ++w) before += __popc(known[w]);
  const int own = before;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  int marked = 0;
  before -= own;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    marked += sums[w];
  }
  for (int w = w_begin; w < w_end; ++w) {
    slot_of[w] = before;
    before += __popc(known[w]);
  }
  __syncthreads();

  bool ok = true;
  int taken = 0;                     // copies waited for
  auto arrived = [&] {
    const bool here = mbar_wait_limited(smem_u32(bar + taken % buffers), (taken / buffers) & 1, kWaitLimit);
    ++taken;
    ok = ok && here;
  };
  bool first_piece = true;
  for (int word0 = 0; word0 < slice_words && 32 * word0 < size;) {
    // ---- the next piece: words that mark kSlots tokens at most (a word marks 32)
    int word1 = slice_words;
    const int slot0 = slot_of[word0];
    if (marked - slot0 > kSlots) {
      if (tid == 0) s_end = word0 + 1;
      __syncthreads();
      for (int w = word0 + 1 + tid; w < slice_words; w += kThreads)
        if (slot_of[w] - slot0 <= kSlots) atomicMax(&s_end, w);      // it may end in front of word w
      __syncthreads();
      word1 = s_end;
    }
    const int slots = (word1 < slice_words ? slot_of[word1] : marked) - slot0;
    if (!first_piece || word1 < slice_words) {      // the rows' first copies were of a slice in one piece
      while (taken < issued) arrived();
      __syncthreads();
      from = 32 * word0;
      tokens = min(32 * word1, size) - from;
      for (int d = 0; d < min(buffers, my_rows); ++d) fetch_next(d);
    }
    first_piece = false;
    auto slot = [&](int k) {        // of a marked token's place; -1 where it is not this piece's
      const int w = k >> 5;
      return k >= 0 && w >= word0 && w < word1 ? slot_of[w] - slot0 + __popc(known[w] & ((1u << (k & 31)) - 1)) : -1;
    };
    for (int i = tid; i < slots; i += kThreads) count[i] = 0, entry[i] = -1;
    for (int w = word0 + tid; w < word1; w += kThreads) {
      int n = slot_of[w] - slot0;
      for (unsigned bits = known[w]; bits; bits &= bits - 1) token[n++] = static_cast<uint16_t>(32 * w + __ffs(bits) - 1);
    }
    __syncthreads();
    auto counted = [&](int k, bool in_prompt) {
      const int i = slot(k);
      if (i < 0) return;
      if (in_prompt) atomicOr(count + i, kPrompt);
      else atomicAdd(count + i, 1u);
    };
    if (listed <= kList)
      for (int i = tid; i < listed; i += kThreads) counted(list[i] & (kSaid - 1), !(list[i] & kSaid));
    else {
      look(h0);
      history(counted);
    }
    const int bias_slot = slot(bias_at), draft_slot = slot(draft_at);
    if (bias_slot >= 0) atomicMax(entry + bias_slot, b0 + tid);
    for (int e = b0 + kThreads + tid; e < b1; e += kThreads) {
      const int i = slot(place(a.bias_ids[e]));
      if (i >= 0) atomicMax(entry + i, e);
    }
    __syncthreads();
    // an entry becomes its bias, by the thread that has the last one of its token
    if (b1 - b0 <= kThreads) {
      const bool last = bias_slot >= 0 && entry[bias_slot] == b0 + tid;
      __syncthreads();
      if (last) {
        entry[bias_slot] = __float_as_int(bias_value);
        atomicOr(count + bias_slot, kBiased);
      }
    } else {
      for (int i = tid; i < slots; i += kThreads)
        if (entry[i] >= 0) {
          entry[i] = __float_as_int(a.bias_values[entry[i]]);
          atomicOr(count + i, kBiased);
        }
    }
    // the drafts that lead to row i, counted in or out: one a thread, whose mask is looked up a row ahead, and those behind them
    unsigned leads = mask_word(0);
    auto drafted = [&](int i, unsigned by) {
      if (draft_slot >= 0 && leads >> (tid & 31) & 1) atomicAdd(count + draft_slot, by);
      for (int j = kThreads + tid; j < (a.masks ? 0 : i + 1); j += kThreads) {
        const int k = slot(place(a.drafts[row0 + j]));
        if (k >= 0) atomicAdd(count + k, by);
      }
    };

    // ---- the rows
    const unsigned* allow = allow_of(0);
    for (int d = 0; d < my_rows; ++d) {
      const int row = row0 + group + d * groups;
      const TIn* x = row_at(d);
      TOut* out = nullptr;
      if constexpr (KEEP) out = static_cast<TOut*>(a.out) + static_cast<size_t>(row) * a.ld_out + lo;
      const bool masked = allow != nullptr;
      if (a.allow)
        for (int w = word0 + tid; w < word1 && 32 * w < size; w += kThreads) may[w] = masked ? allow[w] : ~0u;
      const unsigned next_leads = mask_word(d + 1);
      allow = allow_of(d + 1);
      if (a.drafts) drafted(row - row0, 1u);
      arrived();
      __syncthreads();
      // Vectors as they lie in memory: number n holds the piece's tokens n * N - skew ..  Of the best one so far only where it is and which of its tokens count is
      // kept; which of them it was, is seen at the end.
      const int skew = skew_of(x), vectors = (tokens + skew + N - 1) / N, shift_of = (N - skew) % N;
      const uint4* row_vectors = reinterpret_cast<const uint4*>(buffer + ((taken - 1) % buffers) * buffer_bytes(slice, sizeof(TIn)));
      const uint8_t *known_bytes = reinterpret_cast<const uint8_t*>(known + word0), *may_bytes = reinterpret_cast<const uint8_t*>(may + word0);
      float best = -INFINITY;
      int at = -1;
      unsigned at_plain = 0;
      auto take = [&](int n, unsigned inside, unsigned allowed, unsigned marks) {
        const uint4 u = row_vectors[n];
        const unsigned fine = inside & allowed, plain = fine & ~marks;
        if constexpr (KEEP) {
          float z[N];
#pragma unroll
          for (int j = 0; j < N; ++j) z[j] = fine >> j & 1 ? Vec<TIn>::get(u, j) : -INFINITY;
          store_all<N>(out + from + n * N - skew, z, inside & ~marks);
        }
        const float m = Vec<TIn>::largest(u, keep_of[plain]);
        if (m > best || (at < 0 && plain)) {
          best = m != m ? -INFINITY : m;
          at = n;
          at_plain = plain;
        }
      };
      if (!skew) {
        const int whole = tokens / N;
#pragma unroll 4
        for (int n = tid; n < whole; n += kThreads) {
          const int shift = n * N & 7;
          take(n, kAll, may_bytes[n * N / 8] >> shift, known_bytes[n * N / 8] >> shift);
        }
        if (whole < vectors && tid == kThreads - 1) take(whole, (1u << (tokens - whole * N)) - 1, may_bytes[whole * N / 8] >> (whole * N & 7), known_bytes[whole * N / 8] >> (whole * N & 7));
      } else {
        // the first vector begins ahead of the piece: bits from its token 0 on, moved up; the others N - skew + (n - 1) * N tokens in
#pragma unroll 4
        for (int n = tid; n < vectors; n += kThreads) {
          const int k = n ? shift_of + (n - 1) * N : 0, w = word0 + (k >> 5);
          const unsigned m = __funnelshift_r(may[w], may[w + 1], k & 31), b = __funnelshift_r(known[w], known[w + 1], k & 31);
          const int up = n ? 0 : skew, over = n * N - skew + N - tokens;
          take(n, kAll & kAll << up & (over > 0 ? kAll >> over : kAll), m << up, b << up);
        }
      }
      int id = -1;
      if (at >= 0) {
        const uint4 u = row_vectors[at];
#pragma unroll
        for (int j = N - 1; j >= 0; --j)
          if ((at_plain >> j & 1) && (Vec<TIn>::get(u, j) == best || best == -INFINITY)) id = lo + from + at * N - skew + j;      // (no value above -inf: the first token will do)
      }
      // marked tokens
      const TIn* row_tokens = reinterpret_cast<const TIn*>(row_vectors) + skew - from;
      for (int i = tid; i < slots; i += kThreads) {
        const int k = token[i];
        const bool allowed = may[k >> 5] >> (k & 31) & 1;
        if (!KEEP && !allowed) continue;
        const unsigned c = count[i], n = c & ~(kPrompt | kBiased);
        float z = Vec<TIn>::value(row_tokens[k]);
        if (c & ~kBiased) z = z > 0.f ? __fdiv_rn(z, rho) : __fmul_rn(z, rho);
        z = __fsub_rn(z, __fmul_rn(phi, static_cast<float>(n)));
        if (n) z = __fsub_rn(z, pi);
        if (c & kBiased) z = __fadd_rn(z, __int_as_float(entry[i]));
        if constexpr (KEEP) store_one(out + k, allowed ? z : -INFINITY);
        if (z != z) z = -INFINITY;
        if (allowed && (z > best || id < 0 || (z == best && lo + k < id))) {
          best = z;
          id = lo + k;
        }
      }
      // the warp's best: the largest value, then its lowest token
      const unsigned value = ordered(best, id), top = __reduce_max_sync(0xffffffffu, value);
      const unsigned lowest = __reduce_min_sync(0xffffffffu, value == top ? static_cast<unsigned>(id) : ~0u);
      if (lane == 0 && top) atomicMax(best_of + d, static_cast<unsigned long long>(top) << 32 | (INT_MAX - lowest));
      __syncthreads();      // the row and the counts have been read
      if (d + buffers < my_rows) fetch_next(d + buffers);
      if (a.drafts) drafted(row - row0, ~0u);
      leads = next_leads;
    }
    __syncthreads();
    word0 = word1;
  }
  while (taken < issued) arrived();      // (a slice without tokens)
  if (!ok) *reinterpret_cast<volatile int*>(error) = 1;

  // ---- the slices' best of each row
  if (!a.ids) return;
  __syncwarp();
  cluster_sync_all();
  for (int d = rank + ctas * tid; d < my_rows; d += ctas * kThreads) {
    unsigned long long b = 0;
    for (int c = 0; c < ctas; ++c) b = max(b, peer_load(best_of + d, c));
    a.ids[row0 + group + d * groups] = b ? INT_MAX - static_cast<int>(static_cast<unsigned>(b)) : -1;
  }
  __syncwarp();
  cluster_sync_all();      // no CTA leaves while its best are read
}

template <typename TIn, typename TOut>
int launch(const b200_constrain_args& a, int* error, cudaStream_t st) {
  const auto kernel = constrain_kernel<TIn, TOut>;
  // CTAs of a row: slices of 32 KB; where few rows leave SMs idle, smaller ones.  Two rows on their way where a cluster takes several.
  const long long sms = sm_count();
  int ctas = 1;
  while (ctas < kMostCtas && (static_cast<long long>(a.V) * sizeof(TIn) > static_cast<long long>(ctas) * kSliceBytes || (ctas * static_cast<long long>(a.S) < sms && a.V > 4096 * ctas))) ctas *= 2;
  // groups of a request's rows: three CTAs for each of an SM's two places, or a row a group
  const long long clusters = (6 * sms + ctas - 1) / ctas;
  const int groups = !a.starts ? 1 : static_cast<int>(std::max<long long>((a.T + kRows - 1) / kRows, std::min<long long>((a.T + a.S - 1) / a.S, (clusters + a.S - 1) / a.S)));
  if (groups > 65535) return -1;
  const int slice = ((a.V + ctas - 1) / ctas + 31) / 32 * 32;
  const int buffers = a.starts && a.T > a.S && 2 * buffer_bytes(slice, sizeof(TIn)) <= 2 * kSliceBytes + 32 ? 2 : 1;
  const size_t smem = static_cast<size_t>(buffers) * buffer_bytes(slice, sizeof(TIn)) + (3 * static_cast<size_t>(slice / 32) + 2) * 4;
  static std::atomic<unsigned long long> attr_done{0}, wide_done{0};
  if (!ensure_dynamic_smem(kernel, 192 << 10, &attr_done)) return -3;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -3;
  if (!(wide_done.load() >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return -3;
    wide_done.fetch_or(1ull << (dev & 63));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, groups, a.S + (a.starts && a.ids ? 1 : 0));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, slice, buffers, error) == cudaSuccess ? 0 : -2;
}

}  // namespace

int constrain(const b200_constrain_args& a, int* error, cudaStream_t st) {
  if (a.logits_f32) return !a.out ? launch<float, None>(a, error, st) : a.out_f32 ? launch<float, float>(a, error, st) : launch<float, __nv_bfloat16>(a, error, st);
  return !a.out ? launch<__nv_bfloat16, None>(a, error, st) : a.out_f32 ? launch<__nv_bfloat16, float>(a, error, st) : launch<__nv_bfloat16, __nv_bfloat16>(a, error, st);
}

}  // namespace b200
