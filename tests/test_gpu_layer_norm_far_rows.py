"""GPU tests of layer norm on rows far from 0, whose mean's own rounding is not small beside their
deviations.

Tolerances, u = 2^-24, A and D the means of |x| and of |x - m|: the first sum's m' is off by e0 = 48 u A
(a chain of at most 32 additions in a lane, 10 between lanes and waves, the division).  d = x - m' is
u |x - m'| off.  c, what the differences have in common, is at most e0 and is off by
ec = 48 u mean |d| + u mean |d| <= 49 u (D + e0); d - c by e1 = u (2 |x - m| + e0) + ec.  The variance
mean d^2 - c^2 is off by ev = 52 u (V + e0^2) + 2 e0 ec + ec^2 + u (V + e0^2); rstd by half of ev's share
of V + eps and 4 u, y by those, a unit each for two products and the sum, and the type's rounding."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
U = B.U


def _check(x, w, b, eps, r):
    xd = x.double()
    m = xd.mean(1, keepdim=True)
    dev = (xd - m).abs()
    var = (dev ** 2).mean(1, keepdim=True)
    rs = (var + eps) ** -0.5
    more = 1 + 2.0 ** -7
    e0 = 48 * U * xd.abs().mean(1, keepdim=True)
    ec = 49 * U * (dev.mean(1, keepdim=True) + e0)
    ev = 53 * U * (var + e0 ** 2) + 2 * e0 * ec + ec ** 2
    rel = (0.5 * ev * rs ** 2 + 4 * U) * more
    assert float(rel.max()) < 2.0 ** -10  # (or second-order terms would count)
    assert ((r.mean.double().view(-1, 1) - m).abs() <= (ec + U * m.abs()) * more).all()
    assert ((r.rstd.double().view(-1, 1) - rs).abs() <= rel * rs).all()
    h, wd = (xd - m) * rs, w.double()
    want = h * wd + b.double()
    e1 = U * (2 * dev + e0) + ec
    tol = (wd.abs() * (rs * e1 + h.abs() * (rel + 3 * U))
           + (U + B.unit(r.y.dtype)) * want.abs()) * more
    err = (r.y.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("cols", [7, 96, 511, 768, 1280, 1536, 1600, 4096, 5000, 8192, 9000, 20001])
@pytest.mark.parametrize("mean,deviation", [(1e3, 1.0), (1e4, 1.0), (-1e4, 0.1), (1e4, 0.01),
                                            (-1e6, 3.0)])
def test_far_rows(cols, mean, deviation):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(cols)
    w, b = torch.randn(2, cols, generator=g, device="cuda")
    x = mean + deviation * torch.randn(40, cols, generator=g, device="cuda")
    with B.store_of([w, b], "fp32") as store:
        for eps in (1e-5, 1e-12):
            _check(x, w, b, eps, store.layer_norm(1, x, bias=2, eps=eps))
        # next to ordinary rows, and written over them
        x[::2] = torch.randn(20, cols, generator=g, device="cuda")
        r = store.layer_norm(1, x, bias=2)
        _check(x, w, b, 1e-5, r)
        y = x.clone()
        store.layer_norm(1, y, bias=2, out=r._replace(y=y, mean=r.mean.clone(),
                                                      rstd=r.rstd.clone()))
        assert torch.equal(y, r.y)


@pytest.mark.parametrize("cols", [96, 1280, 3000, 9000])
def test_far_rows_of_bf16(cols):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(cols)
    w, b = torch.randn(2, cols, generator=g, device="cuda").bfloat16().float()
    x = (-3000 + 40 * torch.randn(30, cols, generator=g, device="cuda")).bfloat16()
    with B.store_of([w, b], "bf16") as store:
        for dtype in (torch.float32, torch.bfloat16):
            _check(x, w, b, 1e-5, store.layer_norm(1, x, bias=2, dtype=dtype))


@pytest.mark.parametrize("cols", [5, 64, 700, 5000, 9000])
def test_rows_of_equal_numbers(cols):
    """Their variance is 0, and what a rounded mean leaves is taken off: y is the bias (to the rest of
    49 u of e0 = 48 u |x|, times rstd)."""
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(cols)
    b = torch.randn(cols, generator=g, device="cuda")
    x = (torch.rand(30, 1, generator=g, device="cuda") * 2000 - 1000).expand(30, cols).contiguous()
    with B.store_of([torch.ones(cols, device="cuda"), b], "fp32") as store:
        r = store.layer_norm(1, x, bias=2)
        left = 51 * U * 48 * U * x.abs().double() * 1e-5 ** -0.5
        assert ((r.y.double() - b.double()).abs() <= left + U * b.abs()).all()
        assert (r.rstd.double() * 1e-5 ** 0.5 - 1).abs().max() < 1e-4
        assert ((r.mean - x[:, 0]).abs() <= 2 * U * x[:, 0].abs()).all()
