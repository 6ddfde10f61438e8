// A decode step whose requests share their beginnings: the arguments of its four operations (norm_rope.cu, shared_attention.cu, beam_select.cu,
// beam_reorder.cu) and the index arithmetic that their kernels share.  The latter compiles as plain C++ too, so that what a kernel would
// read and write for given lengths and tables can be checked without a GPU.
#pragma once
#include "tree_step.h"

namespace b200 {
namespace beam {

using tree::kPage;
using tree::Request;

constexpr int kMaxBeams = 32;       // of a request: a lane each
constexpr int kMaxFound = 64;       // candidates of a request
constexpr int kMaxEnds = 1024;
constexpr int kMaxVocab = 393216;

// ---- attention: what its lengths say
struct Lengths {
  const int* starts;
  const int* ctx;
  const int* group_starts;
  const int* shared;
  const int* status;
  int S, T, G, max_blocks, max_rows;      // G is 0 where starts or group_starts do not ascend
  B200_HD Request request(int s) const { return tree::request_of(starts, ctx, s, T, max_blocks, max_rows, status); }
};
// Pieces of 16 rows (token * group + head) of all parts at most: of the requests' own ones by the most rows of each, or where starts ascend (`ordered`) by the step's; and of the groups', which are parts
// only where starts ascend
B200_HD long long most_pieces(const b200_shared_attn_args& a, bool ordered) {
  const long long group = a.q_heads / a.kv_heads, T = a.T, most = a.max_rows < a.T ? a.max_rows : a.T;
  return (ordered ? T * group / 16 + a.S : (most * group + 15) / 16 * a.S) + (a.G ? (T * group + 15) / 16 + a.G : 0);
}
// Whether what they cost fits 32 bits
B200_HD bool costs_fit(const b200_shared_attn_args& a, bool ordered) { return most_pieces(a, ordered) * a.kv_heads <= INT32_MAX / (a.max_blocks + 2ll * tree::kItem); }
// Whether every entry i .. of n + 1 values, a step apart, is in order and within 0 .. most
B200_HD bool ascends(const int* v, int n, int most, int i, int step) {
  bool ok = true;
  for (; i <= n; i += step) ok = ok && v[i] >= 0 && v[i] <= most && (i == n || v[i] <= v[i + 1]);
  return ok;
}

// Rows that read the same keys of the same table: a group's rows and its shared pages, or a request's rows and the keys behind those.
struct Part {
  int row0, rows;      // of the step; no rows: nothing to do
  int k0, k1;          // keys k0 .. k1 - 1, k0 on a page's beginning
  int ctx;             // row i sees keys up to ctx + i, or all where `all`
  int table;           // whose row of the block table
  bool all;
};
// What the requests of group g share: whole pages that its first request has, 0 where there is nothing to share
B200_HD Part group_part(const Lengths& n, int g) {
  Part p = {0, 0, 0, 0, 0, 0, true};
  const int m0 = n.group_starts[g], m1 = n.group_starts[g + 1];
  if (m1 - m0 < 2) return p;
  const int have = n.request(m0).ctx, named = n.shared[g], shared = (have < named ? have : named) / kPage * kPage;
  if (shared <= 0) return p;
  p.row0 = n.starts[m0];
  p.rows = n.starts[m1] - p.row0;
  p.k1 = p.ctx = shared;
  p.table = m0;
  return p;
}
// The group of request s, -1 for none
B200_HD int group_of(const Lengths& n, int s) {
  if (n.G <= 0 || s < n.group_starts[0] || s >= n.group_starts[n.G]) return -1;
  return tree::last_at_most(n.group_starts, n.G, s);
}
// A request's own keys: those behind what it shares
B200_HD Part own_part(const Lengths& n, int s) {
  const Request r = n.request(s);
  Part p = {r.row0, r.rows, 0, r.ctx + r.rows, r.ctx, s, false};
  if (!r.rows) return p;
  const int g = group_of(n, s);
  if (g >= 0) {
    const Part shared = group_part(n, g);
    if (shared.rows && r.ctx >= shared.k1) p.k0 = shared.k1;
  }
  return p;
}
// Part u of the step: the groups' first, then the requests'
B200_HD Part part_of(const Lengths& n, int u) { return u < n.G ? group_part(n, u) : own_part(n, u - n.G); }

// ---- reordering
// The n-th set bit of a mask that has more than n
B200_HD int nth_bit(unsigned mask, int n) {
  for (; n > 0; --n) mask &= mask - 1;
  int b = 0;
  for (; !(mask >> b & 1); ++b) {
  }
  return b;
}
B200_HD int bits_below(unsigned mask, int i) {
  int n = 0;
  for (unsigned m = mask & ((1u << i) - 1); m; m &= m - 1) ++n;
  return n;
}
// Of the new beam i of a request: whose pages it has, and whose last, partly filled page; `parents` are beams of the request, `used` the ones that occur.
struct Heir {
  int parent, page;
};
B200_HD Heir heir_of(const int* parents, int beams, int i) {
  unsigned used = 0, extra = 0, seen = 0;      // extra: beams that are not their parent's first
  for (int j = 0; j < beams; ++j) {
    used |= 1u << parents[j];
    if (seen >> parents[j] & 1) extra |= 1u << j;
    seen |= 1u << parents[j];
  }
  const unsigned childless = ~used & (beams < 32 ? (1u << beams) - 1 : ~0u);
  Heir h = {parents[i], parents[i]};
  if (extra >> i & 1) h.page = nth_bit(childless, bits_below(extra, i));      // as many beams are without a child as are not a first one
  return h;
}

}  // namespace beam

#ifdef __CUDACC__
int norm_rope_kv_write(const b200_norm_rope_args& a, cudaStream_t st);
int64_t shared_attention_workspace(const b200_shared_attn_args& a);
int paged_attention_shared(const b200_shared_attn_args& a, int* error, cudaStream_t st);      // error: pinned, set where a wait ran out
int64_t beam_select_workspace(const b200_beam_select_args& a);
int beam_select(const b200_beam_select_args& a, int* error, cudaStream_t st);
int beam_reorder(const b200_beam_reorder_args& a, cudaStream_t st);
#endif

}  // namespace b200
