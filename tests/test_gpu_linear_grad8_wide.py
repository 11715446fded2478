"""GPU tests of linear gradients where 256 x 256 tiles take the least time (tests/
test_linear_tiles_cpu.py holds that these sizes do): columns, outputs and rows that end inside a
tile, one part and several, both formats and layouts, assigning and adding.

Tolerances as in tests/test_gpu_linear_grad8.py; the products in 64 bits are taken on the GPU."""
import pytest

from gpu_util import torch_mod
from test_gpu_linear_grad8 import U, _inputs, _store

pytestmark = pytest.mark.gpu

# rows, columns, outputs, parts
ONE_PART = [(33, 4099, 5003, 1), (100, 4096, 4096, 1), (333, 4096, 4097, 1), (600, 3000, 5000, 1)]
PARTS = [(2236, 897, 4354, 3), (3367, 3690, 659, 5), (8192, 1280, 5120, 2), (5116, 389, 4393, 7)]
# also more blocks than a round of 256 CUs
SHAPES = ONE_PART + PARTS + [(257, 4100, 4100, 1), (2209, 2523, 1550, 3)]


def _want(store, kept, dy, transposed):
    """(gradient, sum of magnitudes) in 64 bits of the weight and of the bias."""
    torch = torch_mod()
    x = store.restore8(kept, dtype=torch.float32).double()
    d = dy.double()
    dw, mag = x.t() @ d, x.abs().t() @ d.abs()
    if transposed:
        dw, mag = dw.t(), mag.t()
    return (dw, mag), (d.sum(0), d.abs().sum(0))


def _check(store, want, rows, before=None):
    import ttperf
    torch = torch_mod()
    for k, ((w, mag), chain) in enumerate(zip(want, (rows / 16 + 64, rows / 8 + 64))):
        got = store.tensors[k + 1].torch_view(ttperf.BUF_GRAD).reshape(-1)
        unit = 2.0 ** -8 if got.dtype == torch.bfloat16 else U
        w = w.reshape(-1)
        if before:
            w = w + before[k].reshape(-1).double()
        tol = chain * U * mag.reshape(-1) + unit * w.abs() + U * w.abs()
        err = (got.double() - w).abs()
        assert (err <= tol).all(), (k, float((err / tol.clamp(min=1e-300)).max()))


@pytest.mark.parametrize("rows,cols,outs,parts", SHAPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("transposed", [False, True])
def test_wide_tiles(rows, cols, outs, parts, fmt, transposed):
    import ttperf
    torch = torch_mod()
    # rows of dy at an odd pitch and offset in every second case
    x, dy = _inputs(rows, cols, outs, torch.bfloat16, rows + outs, pitch=3 if transposed else 0)
    with _store(cols, outs, "mixed", transposed) as store:
        kept = store.checkpoint8(x, fmt=fmt)
        flat = store.torch_view(ttperf.BUF_GRAD)
        flat.fill_(3.0)
        store.accumulate_linear_grad8(1, kept, dy, bias=2, transposed=transposed)
        want = _want(store, kept, dy, transposed)
        _check(store, want, rows)
        mask = torch.ones(store.total, dtype=torch.bool, device="cuda")
        for i in (1, 2):
            mask[store.offsets[i]:store.offsets[i] + store.tensors[i].numel] = False
        assert (flat[mask] == 3.0).all()  # nothing else of the buffer was written
        first = [store.tensors[i].torch_view(ttperf.BUF_GRAD).clone() for i in (1, 2)]
        store.accumulate_linear_grad8(1, kept, dy, bias=2, transposed=transposed)
        _check(store, want, rows, before=first)
        store.zero_grad()
        store.accumulate_linear_grad8(1, kept, dy, transposed=transposed)  # without the bias
        assert torch.equal(store.tensors[1].torch_view(ttperf.BUF_GRAD), first[0])
        assert not store.has_grad(2)


@pytest.mark.parametrize("rows,cols,outs,parts", ONE_PART[:1] + PARTS[:1])
def test_wide_tiles_into_a_full_precision_store(rows, cols, outs, parts):
    torch = torch_mod()
    x, dy = _inputs(rows, cols, outs, torch.bfloat16, rows)
    with _store(cols, outs, "fp32") as store:
        kept = store.checkpoint8(x)
        store.accumulate_linear_grad8(1, kept, dy, bias=2)
        _check(store, _want(store, kept, dy, False), rows)
