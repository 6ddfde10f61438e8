// The ring of chunks as its warps use it: one that fills and takes, others that take, over barriers that complete, and over some that stop doing so.
#include <stdio.h>

#include <vector>

#include "tree_step.h"

using namespace b200::tree;

static int failed = 0;
#define CHECK(x) do { if (!(x)) { ++failed; printf("line %d: %s (chunks %d, stops %d)\n", __LINE__, #x, chunks, stops); } } while (0)

template <int kRing>
void walk(int chunks, int stops) {      // chunk `stops` never comes
  Ring<kRing> filler, other;
  int full[kRing] = {}, empty[kRing] = {}, lies[kRing];      // phases that have ended; the chunk in a buffer
  int waits_after = 0, drained = 0;
  bool gave_up = false;
  for (int& c : lies) c = -1;
  auto wait_empty = [&](unsigned b, unsigned parity) {
    CHECK(!gave_up);
    CHECK(empty[b] > 0 && parity == static_cast<unsigned>(empty[b] - 1) % 2);      // the phase that the last reader of the buffer ended
    return true;
  };
  auto wait_full = [&](unsigned b, unsigned parity) {
    const bool here = (full[b] & 1) != static_cast<int>(parity);      // the phase of this parity has ended
    if (gave_up) ++waits_after;
    return here;
  };
  auto issue = [&] {
    if (static_cast<int>(filler.issued) >= chunks || !filler.may_issue(wait_empty)) return;
    const int b = filler.issued % kRing, chunk = static_cast<int>(filler.issued);
    CHECK(!gave_up);
    CHECK(lies[b] < 0);                      // nobody still reads what lies there
    if (chunk != stops) lies[b] = chunk, ++full[b];
    ++filler.issued;
  };
  for (int k = 0; k < kRing; ++k) issue();
  for (int c = 0; c < chunks; ++c) {
    const bool a = filler.arrived(wait_full), o = other.arrived(wait_full);
    CHECK(a == o);
    if (!a) {
      gave_up = true;
      continue;      // (rows behind it: no wait is made)
    }
    CHECK(c < stops);
    CHECK(lies[filler.last()] == c && filler.last() == other.last());
    lies[filler.last()] = -1;
    ++empty[filler.last()];
    issue();
  }
  CHECK(filler.ok == (stops >= chunks) && filler.ok == other.ok);
  CHECK(waits_after == 0);
  const int under_way = static_cast<int>(filler.issued - filler.taken);
  filler.drain([&](unsigned b, unsigned) { return ++drained, lies[b] >= 0; });
  CHECK(drained == under_way && filler.taken == filler.issued && drained <= kRing && (filler.ok ? drained == 0 : drained > 0));
}

int main() {
  for (int chunks = 0; chunks < 20; ++chunks)
    for (int stops = 0; stops <= chunks; ++stops) walk<2>(chunks, stops), walk<3>(chunks, stops);
  if (!failed) printf("ok\n");
  return failed != 0;
}
