"""The choice of slices for products of few tiles (csrc/slices.h), on the CPU with made-up GPUs."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "audiocraft.cpp_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "slices.h"
// tiles nk most join one room[1] room[2] ..
int main(int argc, char** argv) {
    auto arg = [&](int i) { return i < argc ? std::atol(argv[i]) : 0; };
    std::printf("%d", act::best_slices(arg(1), (int)arg(2), (int)arg(3), (int)arg(4), arg(5),
                                       [&](int n) { return arg(5 + n); }));
}
"""


@pytest.fixture(scope="module")
def best(tmp_path_factory):
    d = tmp_path_factory.mktemp("slices")
    (d / "s.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I" + CSRC, str(d / "s.cpp"), "-o", str(d / "s")], check=True)

    def run(tiles, nk, most, join, one, room):
        args = [tiles, nk, most, join, one] + list(room)
        return int(subprocess.run([str(d / "s")] + [str(v) for v in args], capture_output=True, text=True, check=True).stdout)

    return run


WHOLE = [148, 74, 44, 36, 26, 22, 18, 18, 14, 10, 8, 8, 8, 8, 8, 8]  # clusters of 1 .. 16 at once


def formula(tiles, nk, most, join, one, room):
    cost = {1: one}
    for n in range(2, min(most, nk) + 1):
        if room[n - 1] > 0:
            cost[n] = -(-tiles // room[n - 1]) * (-(-nk // n) + join)
    return min(cost, key=lambda n: (cost[n], n))


@pytest.mark.parametrize("tiles,nk,most,join,one", [(1, 375, 16, 8, 383), (24, 375, 16, 8, 383), (300, 94, 16, 8, 306),
                                                    (12, 48, 8, 12, 48), (2, 3, 8, 12, 3), (1, 1, 16, 8, 9), (147, 48, 8, 12, 48)])
def test_the_cheapest_number_wins(best, tiles, nk, most, join, one):
    assert best(tiles, nk, most, join, one, WHOLE) == formula(tiles, nk, most, join, one, WHOLE)


def test_sizes_that_cannot_run_are_no_choice(best):
    # one column tile of 375 blocks: sixteen slices, eight where no larger cluster runs, one where none does
    assert best(1, 375, 16, 8, 383, WHOLE) == 16
    assert best(1, 375, 16, 8, 383, WHOLE[:8] + [0] * 8) == 8
    assert best(1, 375, 16, 8, 383, [148] + [0] * 15) == 1
    assert best(1, 375, 16, 8, 383, [148, 74, 0, -1, 26] + [0] * 11) == 5


def test_the_query_says_none_for_sizes_that_do_not_fit():
    # 1 would stand for "one cluster at a time", which a size that cannot be launched then wins with
    text = open(os.path.join(CSRC, "common.cuh")).read()
    body = text[text.index("inline int clusters_at_once"):]
    body = body[:body.index("\n}\n")]
    assert "return 0;" in body and "return 1;" not in body
