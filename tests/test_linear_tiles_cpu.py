"""Host-side checks of how linear gradients are cut into tiles and parts (csrc/linear_tiles.hpp):
which tile the GPU tests' sizes take on the 256 CUs of an MI355X, and that parts cover the rows."""
import os
import random
import subprocess

import pytest

import test_gpu_linear_grad8 as small
import test_gpu_linear_grad8_wide as wide
from conftest import REPO

PROBE = r"""
#include <stdio.h>
#include "linear_tiles.hpp"
int main() {
    unsigned long long rows, cols, outs;
    int bf16;
    while (scanf("%llu %llu %llu %d", &rows, &cols, &outs, &bf16) == 4) {
        const ttp::Cut c = ttp::choose_cut(rows, (uint32_t)cols, (uint32_t)outs, bf16 != 0, 256);
        printf("%d %u %u %u %llu\n", c.wide, c.tiles_a, c.tiles_b, c.parts,
               (unsigned long long)c.per);
    }
}
"""


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    """[(rows, cols, outs, bf16), ...] -> [(wide, tiles_a, tiles_b, parts, per), ...]"""
    d = tmp_path_factory.mktemp("tiles")
    (d / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I",
                    os.path.join(REPO, "tt-perf_amd", "csrc"), "-o", str(d / "probe"),
                    str(d / "probe.cpp")], check=True)

    def run(shapes):
        text = "".join("%d %d %d %d\n" % s for s in shapes)
        out = subprocess.run([str(d / "probe")], input=text, capture_output=True, text=True,
                             check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


def test_the_gpu_tests_reach_both_tiles(cut):
    got = cut([(r, c, o, 1) for r, c, o, _ in wide.SHAPES])
    for (rows, cols, outs, parts), g in zip(wide.SHAPES, got):
        assert g[0] == 1 and g[3] == parts, (rows, cols, outs, g)
    assert {g[3] > 1 for g in got} == {False, True}
    narrow = cut([(*s, 1) for s in small.SHAPES])
    assert not any(g[0] for g in narrow) and {g[3] > 1 for g in narrow} == {False, True}
    planes = cut([(r, c, o, 0) for r, c, o, _ in wide.SHAPES] + [(*s, 0) for s in small.SHAPES])
    assert not any(g[0] for g in planes)


def test_parts_cover_the_rows(cut):
    rng = random.Random(5)
    shapes = [(0, 40, 24, 1), (1, 1, 1, 1), (2 ** 31 - 1, 64, 64, 1), (7, 2 ** 31 - 1, 1, 0)]
    for _ in range(3000):
        shapes.append((int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 14)),
                       int(2 ** rng.uniform(0, 14)), rng.randrange(2)))
    for (rows, cols, outs, _), (w, ta, tb, parts, per) in zip(shapes, cut(shapes)):
        tile = 256 if w else 128
        assert ta == -(-cols // tile) and tb == -(-outs // tile)
        assert per % 32 == 0 and 1 <= parts <= 64
        assert parts * per >= rows and (rows == 0 or (parts - 1) * per < rows)
        assert parts == 1 or per >= 128
