// Host program: how attentions with shared keys are cut.  Arguments, five for each call: query rows, heads,
// kv heads, sequences, groups; a line for each: tile rows of the rests and of the groups, workers, workers
// of a launch of the groups' own.
#include <cstdio>
#include <cstdlib>

#include "dfl_kv4.h"

int main(int argc, char** argv) {
  for (int i = 1; i + 4 < argc; i += 5) {
    const dfl::Kv4SharedCut c = dfl::kv4_shared_cut(std::atoi(argv[i]), std::atoi(argv[i + 1]), std::atoi(argv[i + 2]),
                                                    std::atoi(argv[i + 3]), std::atoi(argv[i + 4]));
    std::printf("%d %d %d %d\n", c.own, c.shared, c.workers, c.shared_workers);
  }
  return 0;
}
