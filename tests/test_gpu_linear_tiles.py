"""GPU tests of the two large tiles of linear products, 256 x 160 and 128 x 256: tiles that end inside
either dimension, sums of one step and of several, whole and partial last steps, sums in parts; and of
a tied output layer's two products.  The tolerances are test_gpu_linear.py's.  (Which tile each size
takes, and in how many parts, tests/test_linear_tile_sizes_cpu.py asserts.)"""
import pytest

import block_util as B
from gpu_util import torch_mod
from test_gpu_linear import _check, _inputs

pytestmark = pytest.mark.gpu

# rows, columns, outputs, transposed
LARGE = [(10091, 456, 792, False), (8268, 4432, 136, False), (2048, 6400, 1600, False),
         (4096, 5120, 1280, False), (11899, 304, 800, False), (16052, 232, 536, True),
         (11023, 3152, 131, True), (12328, 3136, 129, True), (2048, 6400, 1600, True),
         (13410, 368, 523, True)]
WIDE = [(13541, 8, 520, False), (9450, 32, 816, False), (13533, 40, 544, False),
        (11849, 72, 672, False), (13363, 128, 528, False), (14682, 136, 528, False),
        (11065, 7456, 168, False), (299, 8112, 7576, False), (13548, 8, 517, True),
        (13806, 40, 541, True), (13336, 72, 523, True), (9569, 128, 821, True),
        (13366, 136, 543, True)]


@pytest.mark.parametrize("rows,cols,outs,transposed", LARGE + WIDE)
def test_tiles(rows, cols, outs, transposed):
    torch = torch_mod()
    x, w, b = _inputs(rows, cols, outs, "mixed", rows, transposed)
    g = torch.Generator(device="cuda").manual_seed(2)
    with B.store_of([w, b], "mixed") as store:
        y = store.linear(1, x, transposed=transposed)
        _check(y, x, w, transposed=transposed)
        assert torch.equal(store.linear(1, x, transposed=transposed), y)
        for dtype in (torch.bfloat16, torch.float32):
            res = torch.randn(rows, outs, generator=g, device="cuda").to(dtype)
            # into columns of a wider matrix, and over the residual
            out = B.pitched(torch.zeros_like(res), 3, 6, 7.0)
            store.linear(1, x, bias=2, activation="gelu_tanh", residual=res, transposed=transposed,
                         dtype=dtype, out=out)
            _check(out, x, w, b, "gelu_tanh", None, res, transposed)
            assert (out._base[:, :3] == 7).all() and (out._base[:, 3 + outs:] == 7).all()
            store.linear(1, x, bias=2, activation="gelu_tanh", residual=res, transposed=transposed,
                         dtype=dtype, out=res)
            assert torch.equal(res, out)


@pytest.mark.parametrize("rows,cols,outs,transposed", [LARGE[0], LARGE[1], WIDE[2], WIDE[6]])
def test_dropout_behind_the_tiles(rows, cols, outs, transposed):
    torch = torch_mod()
    x, w, b = _inputs(rows, cols, outs, "mixed", rows, transposed)
    res = torch.randn(rows, outs, device="cuda").bfloat16()
    with B.store_of([w, b], "mixed") as store:
        y = store.linear(1, x, bias=2, dropout=(0.1, 5, 3), residual=res, transposed=transposed)
        _check(y, x, w, b, None, (0.1, 5, 3), res, transposed)


@pytest.mark.parametrize("rows", [4097, 129])
def test_a_tied_output_layer(rows):
    """The logits by a table of 50257 tokens, and their gradient back through it: a summed index that is
    no multiple of 8, in contiguous rows and in padded ones."""
    torch = torch_mod()
    vocab, cols = 50257, 768
    x, w, _ = _inputs(rows, cols, vocab, "mixed", rows, True)
    with B.store_of([w], "mixed") as store:
        y = store.linear(1, x, transposed=True)
        _check(y, x, w, transposed=True)
        dy = y
        dx = store.linear_input_grad(1, dy, transposed=True)
        _check(dx, dy, w)
        padded = B.pitched(dy, 0, 7, float("nan"))
        _check(store.linear_input_grad(1, padded, transposed=True), dy, w)
