// The ranges of an attention call's work, walked as its kernel walks them: every tile of every item is taken once, an item that one range does not hold lies in
// consecutive ranges, and the one with its beginning knows in how many.
#include <stdint.h>
#include <stdio.h>

#include <random>
#include <vector>

#include "tree_step.h"

using namespace b200::tree;

static int failed = 0;
#define CHECK(x) do { if (!(x)) { if (++failed < 20) printf("line %d: %s\n", __LINE__, #x); } } while (0)

int main() {
  std::mt19937 rng(2);
  auto pick = [&](int lo, int hi) { return static_cast<int>(lo + rng() % static_cast<uint32_t>(hi - lo + 1)); };
  for (int round = 0; round < 60000; ++round) {
    const int most = pick(0, 3) ? pick(1, 40) : 296, longest = pick(0, 2) == 0 ? 300 : pick(1, 20);
    std::vector<int> tiles(pick(1, 30)), first;
    int N = 0;
    for (int& t : tiles) {
      t = pick(1, longest);
      first.push_back(N);
      N += t + kItem;
    }
    const Ranges r = ranges_of(N, most);
    CHECK(r.n >= 1 && r.n <= most && r.at(0) == 0 && r.at(r.n) == N && r.each >= 1);
    auto item_of = [&](int b) { int i = 0; while (b >= first[i] + tiles[i] + kItem) ++i; return i; };
    struct Part { int range, t0, take; };
    std::vector<std::vector<Part>> of(tiles.size());
    std::vector<int> said(tiles.size(), 0), by(tiles.size(), -1);
    int was = 0;
    for (int c = 0; c < r.n; ++c) {
      int begin = N, end = N, at = 0;
      if (r.at(c) < N) {
        at = item_of(r.at(c));
        begin = snapped(r.at(c), first[at], tiles[at], r.snap);
      }
      if (c + 1 < r.n) {
        const int e = item_of(r.at(c + 1));
        end = snapped(r.at(c + 1), first[e], tiles[e], r.snap);
      }
      CHECK(begin == was && end >= begin);
      was = end;
      int rest = end - begin;
      if (rest <= 0) continue;
      int t0 = begin - first[at] - kItem > 0 ? begin - first[at] - kItem : 0;
      if (t0 == tiles[at]) t0 = 0, ++at;
      int firsts = 0;      // parts without their item's beginning: one place a range has for them
      for (bool more = true; more;) {
        CHECK(at < static_cast<int>(tiles.size()));
        if (at >= static_cast<int>(tiles.size())) break;
        const int take = take_of(t0, tiles[at], &rest);
        CHECK(take >= 1 && t0 + take <= tiles[at]);
        firsts += t0 > 0;
        of[at].push_back({c, t0, take});
        if (rest == 0 && t0 == 0 && take < tiles[at]) {
          said[at] = r.parts(c, end - take, tiles[at]);
          by[at] = c;
        }
        t0 = 0;
        if ((more = rest > 0)) ++at;
      }
      CHECK(rest == 0 && firsts <= 1);
    }
    CHECK(was == N);
    for (size_t i = 0; i < tiles.size(); ++i) {
      int t = 0;
      for (size_t k = 0; k < of[i].size(); ++k) {
        CHECK(of[i][k].t0 == t && of[i][k].range == of[i][0].range + static_cast<int>(k));
        t += of[i][k].take;
      }
      CHECK(t == tiles[i]);
      CHECK(of[i].size() == 1 ? said[i] == 0 : said[i] == static_cast<int>(of[i].size()) && by[i] == of[i][0].range);
    }
  }
  printf("%s\n", failed ? "FAILED" : "ok");
  return failed != 0;
}
