// Which requests of a step have rows, as the operations behind step_maps see it: none that step_maps turned away.
#include <stdio.h>

#include "tree_step.h"

using namespace b200::tree;

int main() {
  const int starts[] = {0, 4, 8, 8, 12}, ctx[] = {16, 16, 3, 0};
  int failed = 0;
  for (int word = 0; word < 8; ++word)
    for (int s = 0; s < 4; ++s) {
      int status[] = {0, 0, 0, 0};
      status[s] = word;
      for (int i = 0; i < 4; ++i) {
        const Request r = request_of(starts, ctx, i, 12, 4, 8, status), plain = request_of(starts, ctx, i, 12, 4, 8);
        const bool away = i == s && (word & 3);      // 4, a parent not in front of its child, turns nobody away
        if (r.rows != (away ? 0 : plain.rows) || r.row0 != (away ? 0 : plain.row0) || r.ctx != (away ? 0 : plain.ctx)) ++failed, printf("status %d of %d: request %d\n", word, s, i);
      }
    }
  if (!failed) printf("ok\n");
  return failed != 0;
}
