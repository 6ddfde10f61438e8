// The index arithmetic of the operations on drafted trees, against buffers of exactly the size their kernels may touch: built with the address and
// undefined-behaviour sanitizers, any read or write beyond them ends the program.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <vector>

#include "tree_step.h"

using namespace b200::tree;

static int failed = 0;
#define CHECK(x) do { if (!(x)) { ++failed; printf("line %d: %s\n", __LINE__, #x); } } while (0)

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return static_cast<int>(lo + rng() % (static_cast<uint32_t>(hi) - static_cast<uint32_t>(lo) + 1u)); };
  const int odd[] = {INT32_MIN, INT32_MIN + 1, -16, -1, 0, 1, 15, 16, 17, INT32_MAX - 15, INT32_MAX - 1, INT32_MAX};
  // requests from any lengths: rows and positions of what is left lie in the buffers
  for (int round = 0; round < 200000; ++round) {
    const int S = pick(1, 4), T = pick(0, 40), blocks = pick(0, 6), most = pick(0, 40);
    std::vector<int> starts(S + 1), ctx(S), rows(T), table(blocks);
    for (int& v : starts) v = pick(0, 9) ? pick(-1, T + 1) : odd[pick(0, 11)];
    for (int& v : ctx) v = pick(0, 9) ? pick(-1, blocks * 16 + 1) : odd[pick(0, 11)];
    for (int& v : table) v = pick(0, 3) ? pick(0, 9) : odd[pick(0, 11)];
    for (int s = 0; s < S; ++s) {
      const Request r = request_of(starts.data(), ctx.data(), s, T, blocks, most);
      CHECK(r.rows >= 0 && r.rows <= most && r.ctx >= 0);
      for (int i = 0; i < r.rows; ++i) rows.at(r.row0 + i) += 1;
      for (int p = 0; p < r.ctx + r.rows; ++p) {
        CHECK(static_cast<size_t>(p >> 4) < table.size());
        const long long at = cache_row(table.data(), p, 7);
        CHECK(at >= -1 && at < 7 * 16);
        CHECK((at >= 0) == (table[p >> 4] >= 0 && table[p >> 4] < 7));
      }
      if (starts[s] >= 0 && starts[s] <= starts[s + 1] && starts[s + 1] <= T && starts[s + 1] - starts[s] <= most && ctx[s] >= 0 && ctx[s] <= 16 * blocks - (starts[s + 1] - starts[s]))
        CHECK(r.rows == starts[s + 1] - starts[s] && r.ctx == ctx[s] && r.row0 == starts[s]);
      else
        CHECK(r.rows == 0);
    }
  }
  // parents: always in front, so that every way up ends
  for (int round = 0; round < 20000; ++round) {
    const int n = pick(1, 30);
    std::vector<int> parents(n);
    for (int& v : parents) v = pick(0, 4) ? pick(-2, n) : odd[pick(0, 11)];
    for (int i = 0; i < n; ++i) {
      int steps = 0;
      for (int j = i; j >= 0; j = parent_of(parents.data(), 0, j)) CHECK(++steps <= n);
      CHECK(parent_of(nullptr, 0, i) == i - 1);
    }
  }
  // sums searched
  for (int round = 0; round < 50000; ++round) {
    const int n = pick(1, 20);
    std::vector<int> v(n + 1);
    for (int i = 1; i <= n; ++i) v[i] = v[i - 1] + (pick(0, 2) ? pick(0, 5) : 0);
    for (int x = 0; x < v[n]; ++x) {
      const int s = last_at_most(v.data(), n, x);
      CHECK(s >= 0 && s < n && v[s] <= x && x < v[s + 1]);
    }
  }
  // pages asked for: every new position has one, and the table a place for it
  for (int round = 0; round < 500000; ++round) {
    const int blocks = pick(0, 9) ? pick(0, 8) : (1 << 27) - 1, words = pick(0, 2);
    int ctx = pick(0, 5) ? pick(0, 140) : odd[pick(0, 11)], n = pick(0, 5) ? pick(0, 140) : odd[pick(0, 11)], held = pick(0, 5) ? pick(0, 9) : odd[pick(0, 11)];
    const int need = pages_asked(ctx, n, held, blocks, words);
    const bool fits = ctx >= 0 && n >= 0 && held >= 0 && held <= blocks && static_cast<long long>(ctx) + n <= 16ll * blocks && ctx <= 16ll * held && (!words || n <= 32 * words);
    CHECK((need >= 0) == fits);
    if (fits) CHECK(held + need <= blocks && 16ll * (held + need) >= static_cast<long long>(ctx) + n && (need == 0 || 16ll * (held + need - 1) < static_cast<long long>(ctx) + n));
    CHECK(rows_asked(n) == (n > 0 ? n : 0));
  }
  printf("%s\n", failed ? "FAILED" : "ok");
  return failed != 0;
}
