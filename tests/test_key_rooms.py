"""Where TokenLogProbs puts the keys that its waves collected together: every place
lies among the keys' own, whatever the waves counted. On the host, from the header
that the kernel uses."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

import nnops_amd

KERNELS = os.path.join(os.path.dirname(nnops_amd.__file__), "csrc", "kernels")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "key_rooms.hpp"

constexpr int kWaves = 8, kRoom = 2048, kWaveRoom = kRoom / kWaves;

// The kernel's loop over what a line of counts gives, with every place looked at.
int main()
{
    int count[kWaves], to[kWaves];
    while (true) {
        for (int& c : count) {
            if (std::scanf("%d", &c) != 1) {
                return 0;
            }
        }
        const int keys = nnops_amd::gather_rooms(count, kWaveRoom, to);
        std::vector<char> taken(kRoom, 0);
        if (keys >= 0) {
            for (int w = 0; w < kWaves; ++w) {
                for (int at = 0; at < count[w]; ++at) {
                    const int place = to[w] + at;
                    if (at >= kWaveRoom || place < 0 || place >= kRoom || place >= keys || taken[place]) {
                        std::printf("wave %d key %d at %d\n", w, at, place);
                        return 1;
                    }
                    taken[place] = 1;
                }
            }
        }
        std::printf("%d\n", keys);
    }
}
"""


@pytest.fixture(scope="module")
def gather(tmp_path_factory):
    at = tmp_path_factory.mktemp("rooms")
    (at / "rooms.cpp").write_text(PROGRAM)
    cxx = shutil.which("g++") or shutil.which("c++")
    subprocess.run([cxx, "-std=c++20", "-Wall", "-Werror", "-I", KERNELS, "-o", str(at / "rooms"),
                    str(at / "rooms.cpp")], check=True)

    def run(rows):
        lines = "\n".join(" ".join(map(str, r)) for r in rows)
        r = subprocess.run([str(at / "rooms")], input=lines, capture_output=True, text=True)
        assert r.returncode == 0, r.stdout
        return [int(x) for x in r.stdout.split()]
    return run


def test_full_rooms_and_empty_ones(gather):
    assert gather([[0] * 8, [256] * 8, [1] * 8, [0, 0, 0, 0, 0, 0, 0, 256], [256, 0, 255, 1, 0, 256, 3, 7]]) == [
        0, 2048, 8, 256, 778]


@pytest.mark.parametrize("counts", [
    [2048] * 8,                              # no threshold: fewer groups than alternatives have a logit
    [1024] * 8,                              # equal logits, 8192 of them
    [4096] * 8, [257] * 8, [512] * 8,        # 32768, and one more than there is room for
    [256] * 7 + [257], [257] + [0] * 7, [0, 0, 0, 4096, 0, 0, 0, 0], [256, 256, 256, 2048, 256, 256, 256, 256],
])
def test_more_than_a_room_moves_nothing(gather, counts):
    assert gather([counts]) == [-1]


def test_random_counts(gather):
    import numpy as np
    r = np.random.RandomState(3)
    rows = [r.randint(0, r.choice([2, 30, 257, 300, 4097]), 8).tolist() for _ in range(400)]
    want = [-1 if max(c) > 256 else sum(c) for c in rows]
    assert gather(rows) == want and {-1} < set(want)
