"""What a merge of the 4-bit cache attention takes for the parts of a segment.
The pair (first, last run) comes from a workspace that needs no initialisation,
so a pair that is no range of this launch's runs must give no parts: its
indices would lead out of the workspace."""
import itertools

import host_cpp

PROGRAM = r"""
#include <cstdio>
#include "kv4_span.cuh"
int main() {
  int first, last, warps;
  while (std::scanf("%d %d %d", &first, &last, &warps) == 3)
    std::printf("%d\n", b2k::attn_parts(first, last, warps));
}
"""


def test_parts_of_spans_good_and_bad(tmp_path):
    values = [-2 ** 31, -2 ** 31 + 1, -7, -1, 0, 1, 2, 5, 1183, 1184, 1185, 1775, 1776, 2 ** 30,
              0x7fc00000, 2 ** 31 - 2, 2 ** 31 - 1]
    cases = list(itertools.product(values, values, [1, 4, 1184, 1776]))
    out = host_cpp.run(tmp_path, PROGRAM, "\n".join("%d %d %d" % c for c in cases)).split()
    assert len(out) == len(cases)
    for (first, last, warps), parts in zip(cases, map(int, out)):
        good = 0 <= first < last < warps       # one run alone has nothing to merge
        assert parts == (last - first + 1 if good else 0), (first, last, warps)
        assert 0 <= parts <= warps
