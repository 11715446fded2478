"""GPU tests of linear gradients from 8-bit inputs at infinities and at the least numbers."""
import math

import pytest

from gpu_util import torch_mod
from test_gpu_linear_grad8 import U, _inputs, _store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_an_infinite_dy_is_infinite_in_the_gradient(dtype, fmt):
    """xhat^T dy with infinities in dy, as 64-bit sums have them: of xhat's sign, NaN where xhat
    is 0 and where infinities of both signs meet."""
    import ttperf
    torch = torch_mod()
    x, dy = _inputs(90, 100, 70, getattr(torch, dtype), 4)
    x[11, 20] = 0.0
    dy[11, 3] = math.inf
    dy[40, 9] = -math.inf
    dy[5, 30], dy[77, 30] = math.inf, math.inf
    dy[60, 50] = math.nan
    with _store(100, 70, "mixed" if dtype == "bfloat16" else "fp32") as store:
        kept = store.checkpoint8(x, fmt=fmt)
        xk = store.restore8(kept, dtype=torch.float32).double().cpu()
        store.accumulate_linear_grad8(1, kept, dy, bias=2)
        dw, db = (store.tensors[i].torch_view(ttperf.BUF_GRAD).double().cpu() for i in (1, 2))
    d = dy.double().cpu()
    for got, want in ((dw.view(100, 70), xk.t() @ d), (db, d.sum(0))):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.isinf(), want.isinf())
        assert torch.equal(got[got.isinf()], want[want.isinf()])


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_least_numbers(dtype):
    """dy so small that an fp32 one's last part is subnormal, against an x that makes the products
    normal: the part is not lost but for what lies below the least bf16, 2^-133 of each dy (the
    other bounds are those of tests/test_gpu_linear_grad8.py)."""
    import ttperf
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(40, 32, generator=g, device="cuda") * 2.0 ** 100
    dy = (torch.randn(40, 24, generator=g, device="cuda") * 2.0 ** -115).to(getattr(torch, dtype))
    with _store(32, 24, "fp32") as store:
        kept = store.checkpoint8(x)
        store.accumulate_linear_grad8(1, kept, dy)
        xk = store.restore8(kept, dtype=torch.float32).double().cpu()
        got = store.tensors[1].torch_view(ttperf.BUF_GRAD).double().cpu().view(32, 24)
    d = dy.double().cpu()
    want, mag = xk.t() @ d, xk.abs().t() @ d.abs()
    lost = 0.0 if dtype == "bfloat16" else 2.0 ** -133 * xk.abs().sum(0)[:, None]
    assert ((got - want).abs() <= (40 / 16 + 64) * U * mag + 2 * U * want.abs() + lost).all()
