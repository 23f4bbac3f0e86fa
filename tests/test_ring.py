"""The consuming side of the kernels' rings of bulk copies (csrc/ring.cuh): the
order of stages and phases, and after a wait that ran out (made here by a wait
that refuses) that nothing more is taken, and that exactly the fills in flight
are waited for before the memory is used for anything else."""
import random

import host_cpp

# For every line "S total fail": a warp with a ring of S stages and `total`
# fills to come, whose wait number `fail` runs out (-1: none does).  As in the
# kernels it issues as far as the ring reaches, then one fill for every one
# taken.  Prints the fills taken, the fills issued and those waited for at the end.
PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "ring.cuh"
int main() {
  int S, total, fail;
  while (std::scanf("%d %d %d", &S, &total, &fail) == 3) {
    b2k::RingUse ring;
    std::vector<int> held(S, -1);             // the fill that each stage holds
    unsigned issued = 0;
    int waits = 0, wrong = 0;
    auto issue = [&] { held[issued % S] = (int)issued; ++issued; };
    while ((int)issued < total && (int)issued < S) issue();
    // phase p of a stage belongs to the fills k with (k / S) % 2 == p
    auto right = [&](int stage, uint32_t phase) {
      if (held[stage] < 0 || (uint32_t)(held[stage] / S & 1) != phase) ++wrong;
    };
    std::printf("taken");
    for (int k = 0; k < total; ++k) {
      const int stage = ring.take(S, [&](int s, uint32_t p) { right(s, p); return waits++ != fail; });
      if (stage < 0) continue;                // the loop goes on, nothing is taken
      std::printf(" %d", held[stage]);
      if ((int)issued < total) issue();
    }
    std::printf(" issued %u drained", issued);
    if (ring.dead)
      ring.drain(issued, S, [&](int s, uint32_t p) { right(s, p); std::printf(" %d", held[s]); return false; });
    std::printf(" wrong %d\n", wrong);
  }
}
"""


def test_a_wait_that_runs_out_leaves_nothing_in_flight(tmp_path):
    rng = random.Random(0)
    cases = [(s, n, f) for s in (1, 2, 3, 4) for n in (0, 1, 2, 3, 4, 5, 9, 23) for f in range(-1, n)]
    cases += [(rng.randint(2, 4), n, rng.randrange(n)) for n in (100, 1000, 3001)]
    lines = host_cpp.run(tmp_path, PROGRAM, "\n".join("%d %d %d" % c for c in cases)).splitlines()
    assert len(lines) == len(cases)
    for (s, n, fail), line in zip(cases, lines):
        taken, rest = line.split("taken")[1].split("issued")
        issued, rest = rest.split("drained")
        drained, wrong = rest.split("wrong")
        taken, drained, issued = [int(x) for x in taken.split()], [int(x) for x in drained.split()], int(issued)
        count = n if fail < 0 else fail
        assert taken == list(range(count))
        assert issued == min(n, count + s)
        # the fill whose wait ran out, and all that were issued after it
        assert drained == ([] if fail < 0 else list(range(count, issued)))
        assert int(wrong) == 0
