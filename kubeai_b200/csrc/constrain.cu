// Penalties, biases and grammar masks on logits, and the greedy choice, in one pass over the rows.
//
//   y = x;  said anywhere: y = y > 0 ? y / rho : y rho;  y -= phi c;  y -= pi where c > 0;  y += bias;  not allowed: -inf;  id = argmax y
//
// A vocabulary's rows are long and what is said about single tokens is short.  A CTA marks the tokens of its part of the vocabulary that the request's lists
// name with a bit each.  The bits' running count gives every such token a slot, where its count, its bias and its number lie: as much shared memory as there
// is to say, whatever the vocabulary.  More tokens than slots: the part is worked on in pieces that have no more.  All of this is done once for the rows of a
// request that the CTA takes.  A row then comes in chunks of 8192 tokens by bulk copies, two or three ahead, from one row into the next; of its vectors eight tokens cost
// a maximum of pairs, marked tokens left out, and the chunk's slots, a thread each, alone need the formula.  A row's drafts are counted in ahead of it and out
// behind it.  Few rows: a cluster of CTAs shares the vocabulary, whose best pairs (value, token) meet through distributed shared memory.  Ties go to the lowest token:
// every comparison prefers it.  Every wait for a copy has a limit, and a warp that gave up makes no other: its CTA has no more copied, sets an error mark and still meets the others.
//
// What bounds it: the lists' chain of look-ups, marks, slots and counts ahead of the rows, which is half of a CTA's time where it has one or two rows (128 rows of 128256
// bf16 logits, 4000 tokens of history each: 25 us, of which the copies need 5; one row 8.1), and for trees the copies in and out behind it (288 rows of 99991 fp32
// logits, kept: 83 us, 2.8 TB/s).  With the formula inside the pass over the vectors, where it ran in nearly every warp for a few of its lanes, and a row over 16 CTAs
// that all read the lists, the 128 rows took 99 us; a thread that takes the marked tokens of its own 32 of a chunk in place of a slot, 34 (and the trees 112); slots' tokens
// found by walking the words in place of being written by who counts them, 28.
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

constexpr int kThreads = 256, kPlaces = 2, kMostCtas = 16, kRows = 256, kAhead = 8, kSlots = 4096;      // kPlaces: CTAs of an SM
constexpr int kGroup = 32, kTokens = kThreads * kGroup;      // tokens that a thread takes of a chunk, and a chunk's
template <typename T>
constexpr int kDepth = sizeof(T) == 2 ? 3 : 2;               // chunks on their way
constexpr int kMostTokens = 393216, kWaitLimit = 1 << 22;
constexpr unsigned kPrompt = 0x80000000u, kBiased = 0x40000000u;      // of a count: said in the prompt, which the repetition penalty alone counts; has a bias
constexpr unsigned kPromptDraft = 1u << 16;      // of a count: one of a tree's drafts that are of the prompt

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

// TIn: the logits; TOut: y kept, or None; LONG: a CTA may have more than kRows rows (the loop for them costs one row 0.3 us of 8.1).  part: tokens of a CTA, a multiple of 32.
template <typename TIn, typename TOut, bool LONG>
__global__ void __launch_bounds__(kThreads, kPlaces)
constrain_kernel(const __grid_constant__ b200_constrain_args a, int part, int* error) {
  constexpr int N = Vec<TIn>::N, kWarps = kThreads / 32, kChunk = kTokens * static_cast<int>(sizeof(TIn)), kRing = kDepth<TIn>;
  constexpr unsigned kAll = (1u << N) - 1;
  constexpr bool KEEP = !std::is_same<TOut, None>::value;
  extern __shared__ __align__(16) uint8_t smem[];
  const int part_words = part / 32;
  unsigned* known = reinterpret_cast<unsigned*>(smem + kRing * kChunk) + 1;      // [-1 .. part_words] the part's tokens that the lists name
  int* slot_of = reinterpret_cast<int*>(known + part_words + 1);                  // [part_words] marked tokens in front of each word
  __shared__ unsigned count[kSlots];               // how often the token was said, with the marks above
  __shared__ int entry[kSlots];                    // the last bias entry, then the bias
  __shared__ uint16_t token[kSlots];               // places in the part, their low 16 bits: a chunk's first place tells the others
  __shared__ unsigned long long best_of[kRows];
  __shared__ uint4 keep_of[1 << N];                // Vec<TIn>::keep of every set of a vector's tokens
  __shared__ int sums[kWarps], s_end;
  __shared__ uint64_t full[kRing], empty[kRing];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = static_cast<int>(cluster_ctarank()), ctas = gridDim.x;
  const int lo = rank * part, size = max(0, min(part, a.V - lo));
  const int s = blockIdx.z, groups = gridDim.y;
  int group = blockIdx.y;      // the first of this CTA's rows, then of its next kRows
  if (tid == 0) {
    for (int b = 0; b < kRing; ++b) {
      mbar_init(smem_u32(full + b), 1);
      mbar_init(smem_u32(empty + b), kWarps);
    }
    fence_mbar_init();
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
  if (a.history) h0 = a.hist_starts[s], h1 = a.hist_starts[s + 1];
  if (a.prompt_lens) prompt = a.prompt_lens[s];
  if (a.bias_starts) b0 = a.bias_starts[s], b1 = a.bias_starts[s + 1];
  if (a.starts) rows = row0 >= 0 && rows >= row0 && rows <= a.T ? rows - row0 : 0;
  h0 = max(h0, 0), h1 = min(h1, a.history_len);
  b0 = max(b0, 0), b1 = min(b1, a.bias_len);
  // The request's rows follow its history: rows in front of this one are of the prompt.  Where there are any, so is all of the history, which leaves the low
  // bits of a count to at most 256 drafts of a tree and those above them to the prompt's; a chain's prompt rows are seen by all rows behind them.
  const int prompt_rows = static_cast<int>(max(0ll, static_cast<long long>(prompt) - max(0, h1 - h0)));
  const bool prompt_apart = a.masks && prompt_rows;
  if (tree::turned_away(a.status, s)) {      // its rows have no choice
    if (!group && a.ids)
      for (int i = rank * kThreads + tid; i < rows; i += ctas * kThreads) a.ids[row0 + i] = -1;
    return;      // (the whole cluster)
  }
  if (group >= rows) return;
  auto rows_from_group = [&] { return min(kRows, (rows - group + groups - 1) / groups); };
  int my_rows = rows_from_group();
  for (int w = tid; w < part_words + 2; w += kThreads) known[w - 1] = 0;
  for (int d = tid; d < kRows; d += kThreads) best_of[d] = 0;
  for (int d = tid; d < 1 << N; d += kThreads) keep_of[d] = Vec<TIn>::keep(d);
  __syncthreads();

  // ---- the rows' tokens [from, from + tokens) of the part, chunk by chunk: chunk c of a row holds its tokens c * kTokens - skew ..
  int from = 0, tokens = size;
  tree::Ring<kRing> ring;              // chunks (every warp takes them all, warp 0 has them copied)
  int f_row = 0, f_chunk = 0;          // the next one to be issued
  auto skew_of = [&](const TIn* p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(TIn) % N); };      // tokens between a 16-byte boundary and p
  auto row_at = [&](int d) { return static_cast<const TIn*>(a.logits) + static_cast<size_t>(row0 + group + d * groups) * a.ld + lo + from; };
  auto chunks_of = [&](int d) { return (tokens + skew_of(row_at(d)) + kTokens - 1) / (kTokens); };
  auto wait_full = [&](unsigned b, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait_limited(smem_u32(full + b), parity, kWaitLimit)) != 0; };
  auto wait_empty = [&](unsigned b, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait_limited(smem_u32(empty + b), parity, kWaitLimit)) != 0; };
  // warp 0: whole 16 bytes by a copy, a row's ragged ends by threads
  auto issue = [&] {
    if (f_row >= my_rows || !tokens) return;
    if (!ring.may_issue(wait_empty)) return;
    const int b = ring.issued % kRing;
    const TIn* p = row_at(f_row);
    const int skew = skew_of(p), first = f_chunk * kTokens - skew;                              // of its tokens
    const int head = first < 0 ? min(tokens, N - skew) : 0, begin = max(first, 0) + head, end = min(first + kTokens, tokens), whole = max(0, end - begin) / N;
    TIn* dst = reinterpret_cast<TIn*>(smem + b * kChunk) - first;      // of token 0
    const bool tail = begin + whole * N + lane < end;
    if (lane < head) dst[lane] = p[lane];
    if (tail) dst[begin + whole * N + lane] = p[begin + whole * N + lane];
    if (lane < head || tail) fence_proxy_async();      // a later copy into this buffer comes behind these stores
    __syncwarp();
    if (lane == 0) {
      __threadfence_block();
      mbar_arrive_expect_tx(smem_u32(full + b), whole * 16);
      if (whole) bulk_load_1d(smem_u32(dst + begin), p + begin, whole * 16, smem_u32(full + b));
    }
    ++ring.issued;
    if (++f_chunk >= chunks_of(f_row)) f_chunk = 0, ++f_row;
  };
  auto left = [&] {      // the warp has read the chunk that arrived last
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(empty + ring.last()));
  };
  int early = 0;
  for (int d = 0; d < my_rows && early < kRing && tokens; ++d) early = min(kRing, early + chunks_of(d));
  if (warp == 0)
    for (int k = 0; k < kRing; ++k) issue();

  // ---- which tokens of the part the lists name.  What a thread takes first of the biases and drafts stays in its registers.
  auto place = [&](int v) { return v >= lo && v < lo + size ? v - lo : -1; };      // in the part
  auto know = [&](int k) {
    if (k >= 0) atomicOr(known + (k >> 5), 1u << (k & 31));
  };
  auto history = [&](auto f) {      // f(place, said in the prompt)
    for (int base = h0; base < h1; base += kAhead * kThreads) {
      int v[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int i = base + e * kThreads + tid;
        v[e] = i < h1 ? a.history[i] : -1;
      }
#pragma unroll
      for (int e = 0; e < kAhead; ++e) f(place(v[e]), base + e * kThreads + tid - h0 < prompt);
    }
  };
  int bias_at = -1, draft_at = -1;
  float bias_value = 0.f;
  if (b0 + tid < b1) bias_at = a.bias_ids[b0 + tid], bias_value = a.bias_values[b0 + tid];
  if (a.drafts && tid < rows) draft_at = a.drafts[row0 + tid];
  auto mask_word = [&](int d) -> unsigned {      // of row d of this CTA's, the one with this thread's draft
    const int i = group + d * groups;
    return !a.drafts || i >= rows ? 0u : !a.masks ? (tid <= i ? ~0u : 0u) : (tid >> 5) < a.words ? static_cast<unsigned>(a.masks[static_cast<size_t>(row0 + i) * a.words + (tid >> 5)]) : 0u;
  };
  auto allow_of = [&](int d) -> const unsigned* {      // its mask's words of the part
    const int i = group + d * groups;
    if (!a.allow || i >= rows) return nullptr;
    const int m = a.allow_rows ? a.allow_rows[row0 + i] : row0 + i;
    return m >= 0 && m < a.allow_count ? reinterpret_cast<const unsigned*>(a.allow) + static_cast<size_t>(m) * a.ld_allow + lo / 32 : nullptr;
  };
  history([&](int k, bool) { know(k); });
  bias_at = place(bias_at);
  draft_at = place(draft_at);
  know(bias_at);
  for (int i = b0 + kThreads + tid; i < b1; i += kThreads) know(place(a.bias_ids[i]));
  know(draft_at);
  if (a.drafts)
    for (int i = kThreads + tid; i < rows; i += kThreads) know(place(a.drafts[row0 + i]));
  __syncthreads();
  // slots: a thread sums some words, one behind the other
  const int per = (part_words + kThreads - 1) / kThreads, w_begin = min(part_words, tid * per), w_end = min(part_words, w_begin + per);
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
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    marked += sums[w];
  }
  for (int w = w_begin; w < w_end; ++w) {
    slot_of[w] = before;
    before += __popc(known[w]);
  }
  __syncthreads();

  for (;;) {      // kRows rows at a time
    for (int word0 = 0; 32 * word0 < size;) {
      // ---- the next piece: words that mark kSlots tokens at most (a word marks 32)
      int word1 = part_words;
      const int slot0 = slot_of[word0];
      if (marked - slot0 > kSlots) {
        if (tid == 0) s_end = word0 + 1;
        __syncthreads();
        for (int w = word0 + 1 + tid; w < part_words; w += kThreads)
          if (slot_of[w] - slot0 <= kSlots) atomicMax(&s_end, w);      // it may end in front of word w
        __syncthreads();
        word1 = s_end;
      }
      const int slots = (word1 < part_words ? slot_of[word1] : marked) - slot0;
      const bool again = LONG && group != static_cast<int>(blockIdx.y);
      if (word0 || word1 < part_words || again) {
        // the first chunks on their way are those of a part in one piece: they are let by
        if (!word0 && !again)
          for (int k = 0; k < early && ring.arrived(wait_full); ++k) left();
        __syncthreads();
        from = 32 * word0;
        tokens = min(32 * word1, size) - from;
        f_row = f_chunk = 0;
        if (warp == 0)
          for (int k = 0; k < kRing; ++k) issue();
      }
      auto slot = [&](int k) {        // of a marked token's place; -1 where it is not this piece's
        const int w = k >> 5;
        return k >= 0 && w >= word0 && w < word1 ? slot_of[w] - slot0 + __popc(known[w] & ((1u << (k & 31)) - 1)) : -1;
      };
      for (int i = tid; i < slots; i += kThreads) count[i] = 0, entry[i] = -1;
      __syncthreads();
      history([&](int k, bool in_prompt) {
        const int i = slot(k);
        if (i < 0) return;
        token[i] = static_cast<uint16_t>(k);      // (whoever else names it writes the same)
        if (in_prompt) atomicOr(count + i, kPrompt);
        else atomicAdd(count + i, 1u);
      });
      const int bias_slot = slot(bias_at), draft_slot = slot(draft_at);
      if (bias_slot >= 0) token[bias_slot] = static_cast<uint16_t>(bias_at), atomicMax(entry + bias_slot, b0 + tid);
      for (int e = b0 + kThreads + tid; e < b1; e += kThreads) {
        const int k = place(a.bias_ids[e]), i = slot(k);
        if (i >= 0) token[i] = static_cast<uint16_t>(k), atomicMax(entry + i, e);
      }
      if (draft_slot >= 0) token[draft_slot] = static_cast<uint16_t>(draft_at);
      if (a.drafts)
        for (int e = kThreads + tid; e < rows; e += kThreads) {
          const int k = place(a.drafts[row0 + e]), i = slot(k);
          if (i >= 0) token[i] = static_cast<uint16_t>(k);
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
      auto count_draft = [&](int slot, int j, unsigned by) {
        if (j >= prompt_rows) atomicAdd(count + slot, by);
        else if (prompt_apart) atomicAdd(count + slot, by * kPromptDraft);
        else atomicOr(count + slot, kPrompt);
      };
      auto drafted = [&](int i, unsigned by) {
        if (draft_slot >= 0 && leads >> (tid & 31) & 1) count_draft(draft_slot, tid, by);
        for (int j = kThreads + tid; j < (a.masks ? 0 : i + 1); j += kThreads) {
          const int k = slot(place(a.drafts[row0 + j]));
          if (k >= 0) count_draft(k, j, by);
        }
      };
      __syncthreads();

      // ---- the rows
      const unsigned* allow = allow_of(0);
      const int allow_words = (a.V - lo - from + 31) / 32;      // from the piece's first on
      for (int d = 0; d < my_rows; ++d) {
        const int i = group + d * groups, skew = skew_of(row_at(d)), chunks = chunks_of(d);
        TOut* out = nullptr;
        if constexpr (KEEP) out = static_cast<TOut*>(a.out) + static_cast<size_t>(row0 + i) * a.ld_out + lo + from;
        const unsigned *may = allow ? allow + word0 : nullptr, *marks = known + word0;
        const unsigned next_leads = mask_word(d + 1);
        allow = allow_of(d + 1);
        if (a.drafts) {
          drafted(i, 1u);
          __syncthreads();
        }
        float best = -INFINITY, at_best = -INFINITY;
        int id = -1, at = 0;               // the best marked token; of the others the best one's vector: its first token's place in the piece, and which of them count
        unsigned at_plain = 0;
        // the masks of a thread's group, looked up a chunk ahead
        unsigned next0 = ~0u, next1 = ~0u;
        auto look_ahead = [&](int k) {
          const int w = k >> 5;              // (-1 where the first group begins ahead of the piece)
          next0 = next1 = ~0u;
          if (!may || k >= tokens) return;
          if (w >= 0) next0 = may[w];
          if (skew && w + 1 < allow_words) next1 = may[w + 1];
        };
        look_ahead(tid * kGroup - skew);
        for (int c = 0; c < chunks; ++c) {
          const int first = c * kTokens - skew, k0 = first + tid * kGroup;      // of the chunk's tokens; of this thread's
          const unsigned may0 = next0, may1 = next1;
          look_ahead(k0 + kTokens);
          // the chunk's slots: those of its tokens, in order
          const int t0 = max(first, 0), t1 = min(first + kTokens, tokens);
          auto slots_ahead = [&](int k) { return k >= tokens ? slots : slot_of[word0 + (k >> 5)] - slot0 + __popc(marks[k >> 5] & ((1u << (k & 31)) - 1)); };
          const int slot_begin = slots_ahead(t0), slot_end = slots_ahead(t1);
          // a thread's first one, from the last warp on, as warp 0 has chunks to issue
          const int mine = slot_begin + kThreads - 1 - tid;
          auto place_of = [&](int n) { return t0 + ((token[n] - (from + t0)) & 0xffff); };      // in the piece
          const int place0 = mine < slot_end ? place_of(mine) : 0;
          unsigned may_first = ~0u;
          if (may && mine < slot_end) may_first = may[place0 >> 5];
          if (!ring.arrived(wait_full)) break;
          const uint4* vectors = reinterpret_cast<const uint4*>(smem + ring.last() * kChunk);
          // a thread's group's bits, then its warp's vectors in the order of memory, each with the bits of the group that it belongs to
          unsigned fine = 0, own = 0, plain = 0;      // allowed ones, ones to be written here, ones that are neither marked nor forbidden
          if (k0 < tokens) {
            const int w = k0 >> 5, over = k0 + kGroup - tokens;
            const unsigned inside = (k0 < 0 ? ~0u << -k0 : ~0u) & (over > 0 ? ~0u >> over : ~0u);
            fine = inside & __funnelshift_r(may0, may1, k0 & 31);
            own = inside & ~__funnelshift_r(marks[w], skew ? marks[w + 1] : 0u, k0 & 31);
            plain = fine & own;
          }
          constexpr int kOwn = kGroup / N;
#pragma unroll
          for (int e = 0; e < kOwn; ++e) {
            const int v = e * 32 + lane, shift = v % kOwn * N, k = first + (warp * 32 * kOwn + v) * N;
            const uint4 u = vectors[warp * 32 * kOwn + v];
            const unsigned here = __shfl_sync(0xffffffffu, plain, v / kOwn) >> shift & kAll;
            if constexpr (KEEP) {
              const unsigned shown = __shfl_sync(0xffffffffu, fine, v / kOwn) >> shift, written = __shfl_sync(0xffffffffu, own, v / kOwn) >> shift & kAll;
              float z[N];
#pragma unroll
              for (int j = 0; j < N; ++j) z[j] = shown >> j & 1 ? Vec<TIn>::get(u, j) : -INFINITY;
              if (written) store_all<N>(out + k, z, written);
            }
            const float top = Vec<TIn>::largest(u, keep_of[here]);
            if (top > at_best || (!at_plain && here)) {
              at_best = top != top ? -INFINITY : top;
              at = k;
              at_plain = here;
            }
          }
          for (int n = mine; n < slot_end; n += kThreads) {
            const int k = n == mine ? place0 : place_of(n), v = k + from;
            const bool allowed = (n == mine || !may ? may_first : may[k >> 5]) >> (k & 31) & 1;
            const unsigned said = count[n], times = said & (prompt_apart ? kPromptDraft - 1 : ~(kPrompt | kBiased));
            float z = Vec<TIn>::value(reinterpret_cast<const TIn*>(vectors)[k - first]);
            if (said & ~kBiased) z = z > 0.f ? __fdiv_rn(z, rho) : __fmul_rn(z, rho);
            z = __fsub_rn(z, __fmul_rn(phi, static_cast<float>(times)));
            if (times) z = __fsub_rn(z, pi);
            if (said & kBiased) z = __fadd_rn(z, __int_as_float(entry[n]));
            if constexpr (KEEP) store_one(out + k, allowed ? z : -INFINITY);
            if (z != z) z = -INFINITY;
            if (allowed && (z > best || id < 0)) best = z, id = lo + v;      // (a thread's slots ascend)
          }
          left();
          if (warp == 0) issue();
        }
        // which token of its vector the best other one is: the first of that value, or the first at all where none is above -inf.  The warp's best ones look.
        __syncwarp();
        const unsigned other = at_plain ? ordered(at_best, 0) : 0u, most = __reduce_max_sync(0xffffffffu, other);
        if (other && other == most && (id < 0 || at_best >= best)) {
          const TIn* x = row_at(d) + at;
          int found = 0;
          for (unsigned bits = at_plain; bits; bits &= bits - 1) {
            found = __ffs(bits) - 1;
            if (at_best == -INFINITY || Vec<TIn>::value(x[found]) == at_best) break;
          }
          found += lo + from + at;
          if (id < 0 || at_best > best || found < id) best = at_best, id = found;
        }
        __syncwarp();
        // the warp's best: the largest value, then its lowest token
        const unsigned value = ordered(best, id), top = __reduce_max_sync(0xffffffffu, value);
        const unsigned lowest = __reduce_min_sync(0xffffffffu, value == top ? static_cast<unsigned>(id) : ~0u);
        if (lane == 0 && top) atomicMax(best_of + d, static_cast<unsigned long long>(top) << 32 | (INT_MAX - lowest));
        if (a.drafts) {
          __syncthreads();      // the counts have been read
          drafted(i, ~0u);
        }
        leads = next_leads;
      }
      __syncthreads();
      word0 = word1;
    }
    if (warp == 0) ring.drain(wait_full);      // no copy is on its way when the CTA ends, where it gave up either
    if (!ring.ok) *reinterpret_cast<volatile int*>(error) = 1;
    // ---- the parts' best of each row
    __syncthreads();
    if (a.ids) {
      if (ctas > 1) cluster_sync_all();
      for (int d = rank + ctas * tid; d < my_rows; d += ctas * kThreads) {
        unsigned long long b = best_of[d];
        for (int c = 0; c < ctas; ++c)
          if (c != rank) b = max(b, peer_load(best_of + d, c));
        a.ids[row0 + group + d * groups] = b ? INT_MAX - static_cast<int>(static_cast<unsigned>(b)) : -1;
      }
      __syncwarp();
      if (ctas > 1) cluster_sync_all();      // no CTA leaves while its best are read
    }
    if (!LONG || rows - group <= kRows * groups) break;
    group += kRows * groups;
    my_rows = rows_from_group();
    __syncthreads();
    for (int d = tid; d < kRows; d += kThreads) best_of[d] = 0;
    __syncthreads();
  }
}

template <typename TIn, typename TOut, bool LONG>
int launch_with(const b200_constrain_args& a, int groups, int* error, cudaStream_t st) {
  const auto kernel = constrain_kernel<TIn, TOut, LONG>;
  const long long places = static_cast<long long>(kPlaces) * sm_count(), each = a.starts ? (a.T + a.S - 1) / a.S : 1;
  int ctas = 1;
  while (ctas < kMostCtas && 2ll * ctas * a.S * groups <= (each > 1 ? 4 : 1) * places && a.V > 4096 * ctas) ctas *= 2;
  const int part = ((a.V + ctas - 1) / ctas + 31) / 32 * 32;
  const size_t smem = kDepth<TIn> * kTokens * static_cast<int>(sizeof(TIn)) + (2 * static_cast<size_t>(part / 32) + 2) * 4;
  static std::atomic<unsigned long long> attr_done{0}, wide_done{0};
  if (!ensure_dynamic_smem(kernel, kDepth<TIn> * kTokens * static_cast<int>(sizeof(TIn)) + (2 * (kMostTokens / 32) + 2) * 4, &attr_done)) return -3;
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
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = pdl_enabled() ? attr : attr + 1;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, part, error) == cudaSuccess ? 0 : -2;
}

template <typename TIn, typename TOut>
int launch(const b200_constrain_args& a, int* error, cudaStream_t st) {
  // A request has one row: as many CTAs as the SMs have places, a row over several of them where that leaves some free (128 rows of 128256 tokens: 28 us
  // over two, 37 over one, 38 over four; one row 8.5 us over 16, 27 over one; with the tables as they were then; now 25 and 8.1).  Several rows: their numbers differ, and most groups of a row end at once, so four
  // times that (16 trees of up to 32 rows of 99991 fp32 logits: 82 us over four CTAs, 96 over one, 100 over two).  More rows than that: groups of several,
  // which read their request's lists once.
  const long long places = static_cast<long long>(kPlaces) * sm_count(), each = a.starts ? (a.T + a.S - 1) / a.S : 1;
  // (and, where requests differ, groups for the longest one there may be, of kRows rows each, as far as a launch has room for so many of every request)
  const long long longest = std::min<long long>((a.T + kRows - 1) / kRows, 65535 / a.S);
  const int groups = static_cast<int>(std::max<long long>(longest, a.S * each <= places ? each : std::min(each, (3 * places + a.S - 1) / a.S)));
  return static_cast<long long>(groups) * kRows < (a.starts ? a.T : 1) ? launch_with<TIn, TOut, true>(a, groups, error, st) : launch_with<TIn, TOut, false>(a, groups, error, st);
}

}  // namespace

int constrain(const b200_constrain_args& a, int* error, cudaStream_t st) {
  if (a.logits_f32) return !a.out ? launch<float, None>(a, error, st) : a.out_f32 ? launch<float, float>(a, error, st) : launch<float, __nv_bfloat16>(a, error, st);
  return !a.out ? launch<__nv_bfloat16, None>(a, error, st) : a.out_f32 ? launch<__nv_bfloat16, float>(a, error, st) : launch<__nv_bfloat16, __nv_bfloat16>(a, error, st);
}

}  // namespace b200
