"""GPU tests of layer norm and its gradients against the formulas in 64 bits.

Tolerances, with u = 2^-24: a row's sum of N numbers is a chain of at most 32 additions in a lane and
10 between lanes and waves (64 bits in rows that are read again): 48 u of the mean magnitude with the
division.  The mean's error d moves (x - m) r by r d, and the variance by d^2 beside its own 50 u, of
which rstd takes half; each further product or sum is one u.  The backward is given mean and rstd,
so h = (x - m) r is 2 u off, g = dy w one, and the means of g and g h 52 and 55 u of their mean
magnitudes.  The weight's and bias's sums are chains of the rows / 2048 of a wave and 40 joins (of
rows that are read again: of a part's rows).  Then one rounding to the type."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
U = B.U


def _inputs(rows, cols, dtype, seed, offset=0.3):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-8, 9, (rows, 1), generator=g, device="cuda").float())
    return (x + offset).to(dtype), torch.randn(rows, cols, generator=g, device="cuda")


def _weights(cols, mode, seed=0):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(2, cols, generator=g, device="cuda") * 0.5
    return [v.to(B.param_dtype(mode)).float() for v in (w[0] + 1, w[1])]


def _check_forward(x, w, b, eps, r):
    torch = torch_mod()
    xd = x.double()
    m = xd.mean(1, keepdim=True)
    var = ((xd - m) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + eps)
    dm = 48 * U * xd.abs().mean(1, keepdim=True)
    assert ((r.mean.double().view(-1, 1) - m).abs() <= dm + 1e-45).all()
    rel = 0.5 * (52 * U + dm * dm * rs * rs) + 4 * U
    assert ((r.rstd.double().view(-1, 1) - rs).abs() <= rel * rs).all()
    wd, bd = (1.0 if w is None else w.double()), (0.0 if b is None else b.double())
    h = (xd - m) * rs
    want = h * wd + bd
    tol = (abs(wd) * (rs * dm + h.abs() * (rel + 4 * U)) + U * want.abs()
           + B.unit(r.y.dtype) * want.abs()) * (1 + 2.0 ** -7) + 1e-38
    err = (r.y.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


def _check_backward(x, dy, w, r, dx, add=None):
    torch = torch_mod()
    xd, wd = x.double(), 1.0 if w is None else w.double()
    rs = r.rstd.double().view(-1, 1)
    h = (xd - r.mean.double().view(-1, 1)) * rs
    g = dy.double() * wd
    want = rs * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    mag = g.abs() + g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True)
    if add is not None:
        want = want + add.double()
    tol = (rs * mag * 64 * U + (U + B.unit(dx.dtype)) * want.abs()) * (1 + 2.0 ** -7) + 1e-38
    err = (dx.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    return h


def _check_sums(store, h, dy, rows, old=None, long_rows=False):
    d = dy.double()
    chain = (rows if long_rows else rows / 2048) + 48
    for k, (want, mag) in enumerate((((d * h).sum(0), (d * h).abs().sum(0)),
                                     (d.sum(0), d.abs().sum(0)))):
        got = B.grad(store, k + 1)
        if old:
            want = want + old[k].double()
        tol = (chain + 4) * U * mag + (B.unit(got.dtype) + U) * (want.abs() + chain * U * mag)
        err = (got.double() - want).abs()
        assert (err <= tol + 1e-38).all(), (k, float((err / tol.clamp(min=1e-300)).max()))


SHAPES = [(1, 1), (1, 2), (3, 7), (257, 384), (9, 511), (64, 512), (5, 513), (33, 1024), (7, 1025),
          (2050, 768), (1000, 1280), (12, 1537), (21, 2048), (4, 2049), (6, 4096), (300, 4097),
          (2, 8192), (3, 8193), (10, 20001)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("mode", ["mixed", "fp32"])
def test_forward_and_backward(rows, cols, dtype, mode):
    import ttperf
    torch = torch_mod()
    dtype = getattr(torch, dtype)
    x, dy = _inputs(rows, cols, dtype, rows + cols)
    dy = dy.to(dtype)
    w, b = _weights(cols, mode)
    with B.store_of([w, b], mode) as store:
        store.torch_view(ttperf.BUF_GRAD).fill_(3.0)
        r = store.layer_norm(1, x, bias=2, eps=1e-5)
        assert r.y.dtype == dtype and r.mean.shape == r.rstd.shape == (rows,)
        _check_forward(x, w, b, 1e-5, r)
        dx = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2)
        h = _check_backward(x, dy, w, r, dx)
        _check_sums(store, h, dy, rows, long_rows=cols > 8192)
        assert [store.has_grad(i) for i in range(4)] == [False, True, True, False]
        assert B.untouched(store, (1, 2), 3.0)
        # a second micro-batch is added, with a gradient that joins; the same inputs, the same bits
        first = [B.grad(store, k).clone() for k in (1, 2)]
        dx2 = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2, add=x)
        _check_backward(x, dy, w, r, dx2, add=x)
        _check_sums(store, h, dy, rows, old=first, long_rows=cols > 8192)
        store.zero_grad()
        again = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2)
        assert torch.equal(again, dx)
        assert all(torch.equal(B.grad(store, k), f) for k, f in zip((1, 2), first))
        assert torch.equal(store.layer_norm(1, x, bias=2, eps=1e-5).y, r.y)


@pytest.mark.parametrize("xt,yt", [("bfloat16", "float32"), ("float32", "bfloat16")])
@pytest.mark.parametrize("cols", [100, 1300, 3000, 9000])
def test_a_result_of_another_type(xt, yt, cols):
    torch = torch_mod()
    xt, yt = getattr(torch, xt), getattr(torch, yt)
    x, dy = _inputs(70, cols, xt, 3)
    dy = dy.to(yt)
    w, b = _weights(cols, "bf16")
    with B.store_of([w, b], "bf16") as store:
        r = store.layer_norm(1, x, bias=2, dtype=yt)
        assert r.y.dtype == yt
        _check_forward(x, w, b, 1e-5, r)
        dx = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2)
        assert dx.dtype == xt
        _check_sums(store, _check_backward(x, dy, w, r, dx), dy, 70, long_rows=cols > 8192)


@pytest.mark.parametrize("cols", [65, 1600, 2500, 8200])
def test_strides_and_places(cols):
    torch = torch_mod()
    x, dy = _inputs(50, cols, torch.float32, 4)
    w, b = _weights(cols, "fp32")
    with B.store_of([w, b], "fp32") as store:
        r = store.layer_norm(1, x, bias=2)
        want = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2, add=dy)
        grads = [B.grad(store, k).clone() for k in (1, 2)]
        for left, right in ((1, 2), (8, 0), (3, 3)):
            xp, dp = B.pitched(x, left, right), B.pitched(dy, right, left)
            out = ttp_result(r, B.pitched(torch.zeros_like(x), left, right, 7.0))
            q = store.layer_norm(1, xp, bias=2, out=out)
            assert torch.equal(q.y, r.y) and torch.equal(q.rstd, r.rstd)
            assert (out.y._base[:, :left] == 7).all() and (out.y._base[:, left + cols:] == 7).all()
            for place in ("dy", "add", "x", "all"):
                xs, ds, ad = xp.clone(), dp.clone(), dp.clone()
                if place == "all":  # the gradient that joins is dy itself
                    ad = ds
                to = {"dy": ds, "add": ad, "x": xs, "all": ds}[place]
                store.zero_grad()
                got = store.layer_norm_backward(1, xs, ds, r.mean, r.rstd, bias=2, add=ad, out=to)
                assert got is to and torch.equal(got, want), place
                assert all(torch.equal(B.grad(store, k), g) for k, g in zip((1, 2), grads))
        y = xp.clone()
        store.layer_norm(1, y, bias=2, out=ttp_result(r, y))  # in the input's place
        assert torch.equal(y, r.y)


def ttp_result(r, y):
    import ttperf
    return ttperf.LayerNorm(y, r.mean.clone(), r.rstd.clone())


def test_without_weight_or_bias():
    torch = torch_mod()
    x, dy = _inputs(30, 200, torch.float32, 5)
    w, b = _weights(200, "fp32")
    with B.store_of([w, b], "fp32") as store:
        r = store.layer_norm(None, x)
        _check_forward(x, None, None, 1e-5, r)
        _check_backward(x, dy, None, r, store.layer_norm_backward(None, x, dy, r.mean, r.rstd))
        assert not any(store.has_grad(i) for i in range(4))
        r = store.layer_norm(1, x)
        _check_forward(x, w, None, 1e-5, r)
        _check_backward(x, dy, w, r, store.layer_norm_backward(1, x, dy, r.mean, r.rstd))
        assert [store.has_grad(i) for i in range(4)] == [False, True, False, False]
        r = store.layer_norm(None, x, bias=2)
        _check_forward(x, None, b, 1e-5, r)
        store.layer_norm_backward(None, x, dy, r.mean, r.rstd, bias=2)
        assert store.has_grad(2)


def test_gradients_are_the_differences():
    """Central differences of sum(dy y) in 64 bits, against the operator's: the formula itself."""
    torch = torch_mod()
    x, dy = _inputs(6, 24, torch.float32, 6)
    w, b = _weights(24, "fp32")
    with B.store_of([w, b], "fp32") as store:
        r = store.layer_norm(1, x, bias=2, eps=1e-3)
        dx = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2)

        def loss(x, w, b):
            m = x.mean(1, keepdim=True)
            v = ((x - m) ** 2).mean(1, keepdim=True)
            return ((x - m) / torch.sqrt(v + 1e-3) * w + b) * dy.double().cpu()

        args = [t.double().cpu() for t in (x, w, b)]
        for k, got in enumerate((dx, B.grad(store, 1), B.grad(store, 2))):
            flat = args[k].reshape(-1)
            for i in range(0, flat.numel(), 5):
                # (a step of 2^-12 of the row's size: truncation and cancellation below 1e-6)
                step = 2.0 ** -12 * float(args[k].reshape(-1).abs().max() if k else
                                          args[0][i // 24].abs().max())
                moved = []
                for sign in (1, -1):
                    a = [t.clone() for t in args]
                    a[k].view(-1)[i] += sign * step
                    moved.append(loss(*a).sum())
                want = float(moved[0] - moved[1]) / (2 * step)
                scale = float(got.abs().max())
                assert abs(float(got.reshape(-1)[i]) - want) <= 1e-4 * scale


def test_special_rows():
    """A row of equal numbers, one with a NaN or an infinity, numbers far from 0: others unmoved."""
    torch = torch_mod()
    for cols in (96, 700, 5000, 8300):
        x, dy = _inputs(8, cols, torch.float32, 7)
        w, b = _weights(cols, "fp32")
        with B.store_of([w, b], "fp32") as store:
            clean = store.layer_norm(1, x, bias=2).y
            x[1], x[2, 5], x[3, -1] = 4.0, float("nan"), float("inf")
            x[4] = x[4] * 0.01 + 1e4
            r = store.layer_norm(1, x, bias=2)
            assert torch.equal(r.y[1], b) and float(r.rstd[1]) == pytest.approx(1e-5 ** -0.5, 1e-6)
            assert r.y[2].isnan().all() and r.y[3].isnan().all()
            assert torch.equal(r.y[5:], clean[5:]) and torch.equal(r.y[0], clean[0])
            row = r._replace(y=r.y[4:5], mean=r.mean[4:5], rstd=r.rstd[4:5])
            _check_forward(x[4:5], w, b, 1e-5, row)
            dx = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2)
            assert dx[2].isnan().all() and dx[3].isnan().all() and dx[4:].isfinite().all()
            assert B.grad(store, 1).isnan().any() and B.grad(store, 2).isfinite().all()


def test_no_rows():
    torch = torch_mod()
    with B.store_of(_weights(64, "mixed"), "mixed") as store:
        x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
        r = store.layer_norm(1, x, bias=2)
        assert r.y.shape == (0, 64) and r.mean.shape == (0,)
        import ttperf
        store.torch_view(ttperf.BUF_GRAD).fill_(5.0)
        store.layer_norm_backward(1, x, x, r.mean, r.rstd, bias=2)
        assert (B.grad(store, 1) == 0).all() and (B.grad(store, 2) == 0).all()
        assert B.untouched(store, (1, 2), 5.0)


@pytest.mark.parametrize("cols", [768, 3001, 9000])
def test_captured(cols):
    import ttperf
    torch = torch_mod()
    x, dy = _inputs(123, cols, torch.float32, 8)
    w, b = _weights(cols, "fp32")
    with B.store_of([w, b], "fp32") as store:
        store.set_stream(torch.cuda.Stream())
        torch.cuda.synchronize()
        r = store.layer_norm(1, x, bias=2)
        dx = store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2)
        store.begin_capture()
        store.zero_grad(set_to_none=True)
        store.layer_norm(1, x, bias=2, out=r)
        store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2, out=dx)
        store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2, add=dx, out=dx)
        graph = store.end_capture()
        for k in range(3):
            x.copy_(_inputs(123, cols, torch.float32, 30 + k)[0])
            torch.cuda.synchronize()
            graph.replay()
            store.sync()
            got = [t.clone() for t in (r.y, r.mean, dx, B.grad(store, 1), B.grad(store, 2))]
            store.zero_grad(set_to_none=True)
            e = store.layer_norm(1, x, bias=2)
            d = store.layer_norm_backward(1, x, dy, e.mean, e.rstd, bias=2)
            d = store.layer_norm_backward(1, x, dy, e.mean, e.rstd, bias=2, add=d)
            want = (e.y, e.mean, d, B.grad(store, 1), B.grad(store, 2))
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(got, want))
        graph.close()
        store.begin_capture()  # whether it assigns or adds is fixed: refused without a call before
        with pytest.raises(ttperf.TTPError):
            store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2, out=dx)
        store.end_capture(discard=True)


def test_refusals():
    import ttperf
    torch = torch_mod()
    x, dy = _inputs(8, 16, torch.float32, 9)
    w, b = _weights(16, "fp32")
    with B.store_of([w, b], "fp32") as store:
        r = store.layer_norm(1, x, bias=2)
        kept = [t.clone() for t in (x, dy, *r)]
        for bad in (dict(index=0), dict(index=9), dict(index=-1), dict(bias=3), dict(eps=-1.0),
                    dict(eps=float("nan")), dict(dtype=torch.float16), dict(x=x.half()),
                    dict(x=x.cpu()), dict(x=x.t()), dict(out=ttp_result(r, r.y.bfloat16()),
                                                         dtype=torch.float32),
                    dict(out=r._replace(mean=r.mean[:4]))):
            a = dict(dict(index=1, x=x, bias=2), **bad)
            with pytest.raises((ValueError, ttperf.TTPError)):
                store.layer_norm(a.pop("index"), a.pop("x"), **a)
        for bad in (dict(index=2), dict(index=0), dict(dy=dy[:4]), dict(dy=dy.half()),
                    dict(mean=r.mean[:4]), dict(rstd=r.rstd.double()), dict(add=dy[:4]),
                    dict(add=dy.bfloat16()), dict(out=dy.bfloat16()),
                    dict(mean=r.mean.cpu())):
            a = dict(dict(index=1, x=x, dy=dy, mean=r.mean, rstd=r.rstd, bias=2), **bad)
            with pytest.raises((ValueError, ttperf.TTPError)):
                store.layer_norm_backward(a.pop("index"), a.pop("x"), a.pop("dy"), a.pop("mean"),
                                          a.pop("rstd"), **a)
        flat = torch.zeros(8 * 16 + 8, device="cuda")
        with pytest.raises(ValueError, match="overlap"):
            store.layer_norm_backward(1, flat[:128].view(8, 16), dy, r.mean, r.rstd, bias=2,
                                      out=flat[8:].view(8, 16))
        # rows that would be paired in another order
        x3 = x.view(2, 4, 16)
        with pytest.raises(ValueError, match="order"):
            store.layer_norm_backward(1, x3, dy.view(2, 4, 16), r.mean.view(4, 2), r.rstd, bias=2)
        assert all(torch.equal(u, v) for u, v in zip((x, dy, *r), kept))
        assert not any(store.has_grad(i) for i in range(4))


def test_a_place_that_is_read_as_another_type():
    """dx in add's place, where dy lies too, of as many bytes in all but other rows."""
    torch = torch_mod()
    rows, cols = 3, 8
    memory = torch.zeros(64, device="cuda")
    dy = memory[:rows * cols].view(rows, cols)  # 96 bytes: 2 x 32 + 32
    add = memory.view(torch.bfloat16).as_strided((rows, cols), (20, 1))  # 2 x 40 + 16
    x, _ = _inputs(rows, cols, torch.bfloat16, 3)
    w, b = _weights(cols, "fp32")
    with B.store_of([w, b], "fp32") as store:
        r = store.layer_norm(1, x, bias=2)
        with pytest.raises(ValueError, match="overlap"):
            store.layer_norm_backward(1, x, dy, r.mean, r.rstd, bias=2, add=add, out=add)
        assert not memory.any() and not store.has_grad(1)
