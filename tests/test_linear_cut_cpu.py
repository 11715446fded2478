"""Host-side checks of how linear products are cut into tiles and parts (csrc/linear_cut.hpp): which
shape the GPU tests' sizes take on the 256 CUs of an MI355X, and that parts cover the summed index."""
import os
import random
import subprocess

import pytest

import test_gpu_linear as gpu
from conftest import REPO

PROBE = r"""
#include <stdio.h>
#include "linear_cut.hpp"
int main() {
    unsigned long long rows, cols, outs;
    int direct, bf16, transposed;
    while (scanf("%llu %llu %llu %d %d %d", &rows, &cols, &outs, &direct, &bf16, &transposed) == 6) {
        const ttp::LinearCut c =
            ttp::choose_linear_cut(rows, cols, outs, direct != 0, bf16 != 0, transposed != 0, 256);
        printf("%d %u %u %u %u\n", (int)c.shape, c.tile_rows, c.tile_outs, c.parts, c.per);
    }
}
"""
THIN, SMALL, WIDE, LARGE, THIN_ANY, ANY = range(6)


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    """[(rows, cols, outs, direct, bf16, transposed), ...] -> [(shape, rows, outs, parts, per)]"""
    d = tmp_path_factory.mktemp("cut")
    (d / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I",
                    os.path.join(REPO, "tt-perf_amd", "csrc"), "-o", str(d / "probe"),
                    str(d / "probe.cpp")], check=True)

    def run(shapes):
        text = "".join("%d %d %d %d %d %d\n" % s for s in shapes)
        out = subprocess.run([str(d / "probe")], input=text, capture_output=True, text=True,
                             check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


def _direct(cols, outs, transposed):
    return cols % 8 == 0 and (transposed or outs % 8 == 0)


def test_the_gpu_tests_reach_every_shape_and_parts(cut):
    shapes = [(r, c, o, int(_direct(c, o, tr)), 1, tr) for tr in (0, 1)
              for r, c, o in [*gpu.SHAPES, *[s[:3] for s in gpu.LARGER if s[3] != "fp32"]]]
    got = cut(shapes)
    assert {g[0] for g in got} == {THIN, SMALL, WIDE, LARGE, THIN_ANY, ANY}
    assert {(g[0], g[3] > 1) for g in got} >= {(THIN, False), (THIN, True), (SMALL, False),
                                               (SMALL, True), (ANY, False), (ANY, True),
                                               (THIN_ANY, False), (THIN_ANY, True)}
    full = cut([(r, c, o, 0, 0, 0) for r, c, o in gpu.SHAPES])
    assert {(g[0], g[3] > 1) for g in full} == {(s, p) for s in (THIN_ANY, ANY)
                                                for p in (False, True)}


def test_parts_cover_the_summed_index(cut):
    rng = random.Random(1)
    shapes = []
    for _ in range(3000):
        size = [int(2 ** rng.uniform(0, 17)) for _ in range(3)]
        direct = rng.randrange(2)
        shapes.append((*size, direct, 1 if direct else rng.randrange(2), rng.randrange(2)))
    for s, (shape, tile_rows, tile_outs, parts, per) in zip(shapes, cut(shapes)):
        rows, cols, outs, direct, bf16, _ = s
        step = 32 if shape in (WIDE, THIN_ANY, ANY) else 64
        assert (shape in (THIN_ANY, ANY)) == (not direct) and per % step == 0, s
        assert 1 <= parts <= 32 and (parts - 1) * per < cols <= parts * per, (s, parts, per)
        if parts > 1:  # parts of three steps or more, of few tiles
            assert per >= 3 * step
            tiles = -(-rows // tile_rows) * -(-outs // tile_outs)
            assert tiles < (4 if shape == THIN_ANY else 3) * 256
