// A verification step of drafted tokens: the arguments of its four operations (step_maps.cu, tree_attention.cu, constrain.cu,
// tree_accept.cu) and the index arithmetic that their kernels share.  The latter compiles as plain C++ too, so that what a kernel would
// read and write for given lengths and tables can be checked without a GPU.
//
// A step has T rows.  Request s owns rows starts[s] .. starts[s + 1] - 1, its tokens of this step, and has ctx[s] tokens in the paged cache
// in front of them.  Row i of a request lies in the cache at position ctx + i; its place in the sequence is ctx + its depth in the tree.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#include <cuda_runtime.h>
#define B200_HD __host__ __device__ __forceinline__
#else
#define B200_HD inline
#endif

#include "../../include/b200engine.h"

namespace b200 {
namespace tree {

constexpr int kPage = 16;             // tokens of a page
constexpr int kMaxRequests = 8192;    // of a step_maps call: their offsets lie in shared memory
constexpr int kMaxWords = 8;          // words of an ancestor mask: trees of up to 256 rows
constexpr int kMaxTree = 2048;        // rows of a request that tree_accept walks
constexpr int kMaxRows = 1 << 30;     // of a step, or entries of a list: an index may run past the end by the threads of a launch
constexpr int kMaxSaid = 1 << 29;     // tokens of all histories: a count shares its word with two marks

struct Request {
  int row0, rows, ctx;
};

// Whether step_maps gave request s no slots, so that its rows have no K and V in the cache and its table behind the pages it holds names anybody's.
B200_HD bool turned_away(const int* status, int s) { return status && (status[s] & 3); }

// The rows of request s as the device's lengths have them; no rows where they do not describe one: lengths out of order, rows behind T, more
// rows than `most`, or more tokens than its row of the block table has pages for; nor where step_maps turned it away.
B200_HD Request request_of(const int* starts, const int* ctx, int s, int T, int max_blocks, int most, const int* status = nullptr) {
  const int a = starts[s], b = starts[s + 1], c = ctx[s];
  const bool ok = !turned_away(status, s) && a >= 0 && b >= a && b <= T && b - a <= most && c >= 0 && static_cast<long long>(c) + (b - a) <= static_cast<long long>(max_blocks) * kPage;
  Request r;
  r.row0 = ok ? a : 0;
  r.rows = ok ? b - a : 0;
  r.ctx = ok ? c : 0;
  return r;
}

// The cache row (page * 16 + offset) of a position, -1 where the table names a page that the cache does not have.
B200_HD long long cache_row(const int* table, int pos, long long num_pages) {
  const int page = table[pos >> 4];
  return page >= 0 && page < num_pages ? static_cast<long long>(page) * kPage + (pos & 15) : -1;
}

// The slot of a position on a page of this number; -1, which is written nowhere, where the number is no page's.
B200_HD int slot_on(int page, int pos) { return page >= 0 && page <= INT32_MAX / kPage - 1 ? page * kPage + (pos & 15) : -1; }

// A parent counts where it lies in front of its child; every other number stands for the request's last token in the cache (-1).
B200_HD int parent_of(const int* parents, int row0, int i) {
  if (!parents) return i - 1;
  const int p = parents[row0 + i];
  return p >= 0 && p < i ? p : -1;
}

// The last index of the n + 1 ascending values v whose value is at most x; v[0] <= x.
B200_HD int last_at_most(const int* v, int n, int x) {
  int lo = 0, hi = n + 1;      // v[lo] <= x < v[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---- the ranges that the work of an attention call is cut into.  All items' costs, in tiles of keys, lie one behind the other; range c begins at c * each + min(c, more).  An
// item that begins at g0 has its tile t at g0 + kItem + t.
constexpr int kItem = 2;      // what an item costs besides its tiles: its queries' trip and its rows' way out
constexpr int kSnap = 3;      // a range does not end within this many tiles of an item's ends, or an eighth of its length
constexpr int kLeast = 2;     // a range's cost at least
struct Ranges {
  int n, each, more, snap;
  B200_HD int at(int c) const { return c * each + (c < more ? c : more); }
  // in how many ranges from c on lies an item of which c has the beginning, but not all: the first tile at g, and how many tiles
  B200_HD int parts(int c, int g, int tiles) const {
    const int x = g + tiles - snap - 1;      // a range that begins in front of it, or there, has the last tiles
    const int last = x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each;
    return (last < n - 1 ? last : n - 1) - c + 1;
  }
};
B200_HD Ranges ranges_of(int cost, int most) {
  Ranges r;
  r.n = cost / kLeast < 1 ? 1 : cost / kLeast < most ? cost / kLeast : most;
  r.each = cost / r.n;
  r.more = cost - r.each * r.n;
  r.snap = r.each / 8 < kSnap ? r.each / 8 : kSnap;
  return r;
}
// the beginning b of a range as it is moved to a tile of the item that begins at g0, its ends among them
B200_HD int snapped(int b, int g0, int tiles, int snap) {
  const int t = b - g0 - kItem;
  return t <= snap ? g0 : g0 + kItem + (tiles - t <= snap ? tiles : t);
}
// The tiles from t0 on of an item that a range takes, which has *rest left, and what is left behind them
B200_HD int take_of(int t0, int tiles, int* rest) {
  const int start = t0 ? 0 : kItem, all = start + tiles - t0, take = *rest >= all ? tiles - t0 : *rest - start;
  *rest -= *rest < all ? *rest : all;
  return take;
}

// The chunks of a ring of `kRing` buffers, in order: which buffer and phase each one's waits are for.  wait(buffer, parity) says whether it came; one that did not
// ends the ring: no buffer is filled again, no chunk behind it is taken, and no other wait is made but those of drain.
template <int kRing>
struct Ring {
  unsigned issued = 0, taken = 0;
  bool ok = true;
  // whether the next chunk's buffer may be filled: what lay there has been read
  template <typename Wait>
  B200_HD bool may_issue(Wait wait) {
    if (ok && issued >= kRing) ok = wait(issued % kRing, (issued / kRing + 1) & 1);
    return ok;
  }
  // whether the next chunk has come
  template <typename Wait>
  B200_HD bool arrived(Wait wait) {
    if (ok) ok = wait(taken % kRing, taken / kRing & 1);
    taken += ok;
    return ok;
  }
  B200_HD int last() const { return static_cast<int>((taken - 1) % kRing); }      // buffer of the chunk that came last
  // a bounded wait more for every chunk still on its way
  template <typename Wait>
  B200_HD void drain(Wait wait) {
    for (; taken != issued; ++taken) wait(taken % kRing, taken / kRing & 1);
  }
};

// What a request asks of step_maps: rows (never negative), and pages beyond those it holds; -1 pages where its lengths do not fit.
B200_HD int rows_asked(int n) { return n > 0 ? n : 0; }
B200_HD int pages_asked(int ctx, int n, int held, int max_blocks, int words) {
  if (ctx < 0 || n < 0 || held < 0 || held > max_blocks) return -1;
  if (static_cast<long long>(ctx) + n > static_cast<long long>(max_blocks) * kPage) return -1;
  if (ctx > static_cast<long long>(held) * kPage) return -1;
  if (words > 0 && n > 32 * words) return -1;
  const int all = static_cast<int>((static_cast<long long>(ctx) + n + kPage - 1) / kPage);
  return all > held ? all - held : 0;
}

}  // namespace tree

#ifdef __CUDACC__
int step_maps(const b200_step_maps_args& a, cudaStream_t st);
int64_t tree_attention_workspace(const b200_tree_attn_args& a);
int paged_attention_tree(const b200_tree_attn_args& a, int* error, cudaStream_t st);      // error: pinned, set where a wait ran out
int constrain(const b200_constrain_args& a, int* error, cudaStream_t st);
int tree_accept(const b200_tree_accept_args& a, cudaStream_t st);
#endif

}  // namespace b200
