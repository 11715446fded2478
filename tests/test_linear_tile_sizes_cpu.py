"""Host-side checks that the sizes of test_gpu_linear_tiles.py take the tiles and parts they are there
for (csrc/linear_cut.hpp, on the 256 CUs of an MI355X)."""
import test_gpu_linear_tiles as gpu
from test_linear_cut_cpu import ANY, LARGE, WIDE, cut  # noqa: F401  (cut: a fixture)


def _reached(cut, sizes):  # noqa: F811
    """{(shape, transposed, parts or one, steps of the last part up to 4, ragged in rows, in outputs,
    in the last step)}"""
    got = set()
    for (rows, cols, outs, tr), (shape, m, n, parts, per) in zip(
            sizes, cut([(r, c, o, 1, 1, int(tr)) for r, c, o, tr in sizes])):
        step = 32 if shape == WIDE else 64
        last = cols - (parts - 1) * per
        got.add((shape, tr, parts > 1, min(-(-last // step), 4), rows % m != 0, outs % n != 0,
                 last % step != 0))
    return got


def test_the_large_tile(cut):  # noqa: F811
    got = _reached(cut, gpu.LARGE)
    assert {g[0] for g in got} == {LARGE}
    for tr in (False, True):
        for parts in (False, True):
            some = [g for g in got if g[1:3] == (tr, parts)]
            assert any(g[4] and g[5] for g in some) and any(g[6] for g in some), (tr, parts)
        assert any(not g[6] for g in got if g[1] == tr)


def test_the_wide_tile(cut):  # noqa: F811
    got = _reached(cut, gpu.WIDE)
    assert {g[0] for g in got} == {WIDE}
    for tr in (False, True):
        whole = [g for g in got if g[1:3] == (tr, False)]
        assert {g[3] for g in whole} == {1, 2, 3, 4}
        assert any(g[4] and g[5] for g in whole) and {g[6] for g in whole} == {False, True}
    # (transposed products are never cut into parts of this tile)
    assert {g[5] for g in got if g[2]} == {True} and (WIDE, False, True) in {g[:3] for g in got}


def test_a_tied_output_layer(cut):  # noqa: F811
    assert cut([(4097, 768, 50257, 1, 1, 1)])[0][0] == WIDE
    assert cut([(4097, 50257, 768, 0, 1, 0)])[0][0] == ANY
