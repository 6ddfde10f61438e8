// The bound on what all parts of a shared attention cost, against the parts themselves: rows in order, and rows that are several requests'.
#include <stdio.h>

#include <algorithm>
#include <random>
#include <vector>

#include "beam_step.h"

using namespace b200;

#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

static int check(unsigned seed) {
  std::mt19937 rng(seed);
  auto in = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  b200_shared_attn_args a = {};
  a.S = in(1, 40), a.G = in(0, 6), a.T = in(1, 300), a.max_blocks = in(1, 9), a.max_rows = in(1, 200), a.kv_heads = in(1, 3), a.q_heads = a.kv_heads << in(0, 3);
  const int group = a.q_heads / a.kv_heads;
  const bool ordered = in(0, 1);
  std::vector<int> starts(a.S + 1), ctx(a.S), groups(a.G + 1), shared(a.G + 1);
  for (int& v : starts) v = in(0, a.T);
  for (int& v : groups) v = in(0, a.S);
  for (int& v : ctx) v = in(0, 100);
  for (int& v : shared) v = in(0, 100);
  std::sort(groups.begin(), groups.end());
  if (ordered) std::sort(starts.begin(), starts.end());
  const bool ascends = beam::ascends(starts.data(), a.S, a.T, 0, 1);
  CHECK(!ordered || ascends);
  const beam::Lengths n = {starts.data(), ctx.data(), groups.data(), shared.data(), nullptr, a.S, a.T, ascends ? a.G : 0, a.max_blocks, a.max_rows};
  long long pieces = 0, cost = 0;
  for (int u = 0; u < n.G + a.S; ++u) {
    const beam::Part p = beam::part_of(n, u);
    const long long some = (static_cast<long long>(p.rows) * group + 15) / 16;
    pieces += some;
    cost += some * ((p.k1 - p.k0 + 15) / 16 + tree::kItem) * a.kv_heads;      // as narrow items of 16 rows, of which no form has more
  }
  CHECK(pieces <= beam::most_pieces(a, false));
  if (ascends) CHECK(pieces <= beam::most_pieces(a, true));
  for (int o = 0; o < 1 + ascends; ++o) {
    CHECK(cost <= beam::most_pieces(a, o) * a.kv_heads * (a.max_blocks + 2 * tree::kItem));
    CHECK(beam::costs_fit(a, o));
  }
  return 0;
}

int main() {
  for (unsigned seed = 0; seed < 20000; ++seed)
    if (check(seed)) return printf("seed %u\n", seed), 1;
  puts("ok");
  return 0;
}
