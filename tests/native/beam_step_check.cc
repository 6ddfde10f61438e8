// The index arithmetic of a step whose requests share their beginnings, for lengths that fit and lengths that do not: what a kernel would read lies in its buffers.
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <vector>

#include "beam_step.h"

using namespace b200;

#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

static int check_parts(unsigned seed) {
  std::mt19937 rng(seed);
  auto in = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const int S = in(0, 9), G = in(0, 5), T = in(0, 40), max_blocks = in(0, 12), max_rows = in(0, 12);
  const bool wild = in(0, 1);
  std::vector<int> starts(S + 1), ctx(S + 1), groups(G + 1), shared(G + 1), status(S + 1, 0);
  for (int& v : starts) v = wild ? in(-3, T + 5) : in(0, T);
  for (int& v : groups) v = wild ? in(-2, S + 2) : in(0, S);
  if (!wild || in(0, 1)) std::sort(starts.begin(), starts.end()), std::sort(groups.begin(), groups.end());
  for (int& v : ctx) v = wild ? in(-5, 230) : in(0, 150);
  for (int& v : shared) v = wild ? in(-40, 300) : in(0, 160);
  if (wild) for (int& v : status) v = in(0, 4);
  const bool ordered = G > 0 && beam::ascends(groups.data(), G, S, 0, 1) && beam::ascends(starts.data(), S, T, 0, 1);
  bool sliced = G > 0;
  for (int i = 0; i < 4 && sliced; ++i) sliced = beam::ascends(groups.data(), G, S, i, 4) && beam::ascends(starts.data(), S, T, i, 4);
  CHECK(sliced == ordered);      // as a kernel's threads look at it
  const beam::Lengths n = {starts.data(), ctx.data(), groups.data(), shared.data(), status.data(), S, T, ordered ? G : 0, max_blocks, max_rows};
  std::vector<int> of_group(T, 0);
  for (int u = 0; u < n.G + S; ++u) {
    const beam::Part p = beam::part_of(n, u);
    CHECK(p.rows >= 0);
    if (!p.rows) continue;
    CHECK(p.row0 >= 0 && p.row0 + p.rows <= T);
    CHECK(p.table >= 0 && p.table < S);
    CHECK(p.k0 >= 0 && p.k0 % beam::kPage == 0 && p.k1 > p.k0 && p.k1 <= max_blocks * beam::kPage);
    CHECK(p.all == (u < n.G));
    if (p.all) {
      CHECK(p.k0 == 0 && p.k1 % beam::kPage == 0);
      for (int t = p.row0; t < p.row0 + p.rows; ++t) CHECK(of_group[t]++ == 0);      // a row is one group's
    } else {
      CHECK(p.k0 <= p.ctx && p.k1 == p.ctx + p.rows);
      if (p.k0) {      // the group's part has all rows of the request, and the keys in front
        const int g = beam::group_of(n, u - n.G);
        CHECK(g >= 0 && g < n.G);
        const beam::Part q = beam::group_part(n, g);
        CHECK(q.k1 == p.k0 && q.row0 <= p.row0 && q.row0 + q.rows >= p.row0 + p.rows);
      }
    }
  }
  return 0;
}

static int check_heirs(unsigned seed) {
  std::mt19937 rng(seed);
  const int B = std::uniform_int_distribution<int>(1, 32)(rng);
  std::vector<int> parents(B);
  for (int& p : parents) p = std::uniform_int_distribution<int>(0, B - 1)(rng);
  std::vector<int> owners(B, 0);
  for (int i = 0; i < B; ++i) {
    const beam::Heir h = beam::heir_of(parents.data(), B, i);
    CHECK(h.parent == parents[i] && h.page >= 0 && h.page < B);
    CHECK(owners[h.page]++ == 0);                                       // a page has one owner
    bool first = true;
    for (int j = 0; j < i; ++j) first = first && parents[j] != parents[i];
    CHECK(first == (h.page == h.parent));
    if (!first) CHECK(std::find(parents.begin(), parents.end(), h.page) == parents.end());      // and what is copied over is nobody's source
  }
  return 0;
}

int main() {
  for (unsigned seed = 0; seed < 20000; ++seed)
    if (check_parts(seed) || check_heirs(seed)) return printf("seed %u\n", seed), 1;
  puts("ok");
  return 0;
}
