"""GPU tests of linear products against products in 64 bits.

Tolerances, u = 2^-24: bf16 products are exact, sums are fp32 chains of cols / 16 matrix instructions
of 16 products and the parts' additions: (cols / 16 + 64) u of the sum of magnitudes.  Of fp32
operands' products six of nine parts are taken (what is left out: 2^-22 of the product), which are six
chains of that length in one: 6 (cols / 16) + 64.  GELU's slope is at most 1.13, its own error
5e-7 of its argument (the distribution function's 2e-7, the exponential's and the reciprocal's units).
Each of bias, factor and residual is one rounding, then one to the type."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
U = B.U


def _inputs(rows, cols, outs, mode, seed, transposed=False):
    torch = torch_mod()
    t = B.param_dtype(mode)
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-4, 5, (rows, 1), generator=g, device="cuda").float())
    shape = (outs, cols) if transposed else (cols, outs)
    w = torch.randn(shape, generator=g, device="cuda") * cols ** -0.5
    b = torch.randn(outs, generator=g, device="cuda")
    return x.to(t), w.to(t).float(), b.to(t).float()


def _act(z, activation):
    torch = torch_mod()
    if activation == "relu":
        return z.clamp(min=0)
    if activation == "gelu":
        return z * torch.special.ndtr(z)
    if activation == "gelu_tanh":
        return z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    return z


def _check(y, x, w, b=None, activation=None, dropout=None, residual=None, transposed=False):
    torch = torch_mod()
    xd, wd = x.double(), w.double()
    wd = wd.t().contiguous() if transposed else wd
    cols = x.shape[-1]
    z, mag = xd @ wd, xd.abs() @ wd.abs()
    six = x.dtype == torch.float32
    tol = ((6 if six else 1) * cols / 16 + 64) * U * mag + (2.0 ** -22 if six else 0) * mag
    if b is not None:
        z = z + b.double()
        tol = tol + U * z.abs()
    want = _act(z, activation)
    if activation in ("gelu", "gelu_tanh"):
        tol = 1.13 * tol + 5e-7 * z.abs()
    if dropout:
        keep = torch.from_numpy(B.kept(*y.shape, *dropout)).cuda()
        t = B.threshold(dropout[0])
        f = 65536.0 / (65536.0 - t)
        want, tol = torch.where(keep, want * f, 0.0), torch.where(keep, (tol + 2 * U * want.abs()) * f, 0.0)
    if residual is not None:
        want = want + residual.double()
        tol = tol + U * want.abs()
    tol = tol + (B.unit(y.dtype) + U) * (want.abs() + tol)
    err = (y.double() - want).abs()
    assert (err <= tol + 1e-38).all(), float((err / tol.clamp(min=1e-300)).max())


SHAPES = [(1, 1, 1), (1, 8, 16), (1, 768, 1000), (2, 33, 7), (3, 1280, 640), (5, 64, 130),
          (8, 250, 65), (15, 511, 129), (16, 2048, 384), (17, 96, 33), (31, 40, 1025),
          (64, 64, 64), (100, 65, 257), (128, 128, 128), (129, 31, 127), (200, 384, 512),
          (257, 384, 160), (300, 200, 1000), (1000, 72, 96), (513, 640, 300)]


@pytest.mark.parametrize("rows,cols,outs", SHAPES)
@pytest.mark.parametrize("mode", ["mixed", "fp32"])
@pytest.mark.parametrize("transposed", [False, True])
def test_products(rows, cols, outs, mode, transposed):
    torch = torch_mod()
    x, w, b = _inputs(rows, cols, outs, mode, rows + cols + outs, transposed)
    g = torch.Generator(device="cuda").manual_seed(1)
    res = torch.randn(rows, outs, generator=g, device="cuda").to(x.dtype)
    with B.store_of([w, b], mode) as store:
        y = store.linear(1, x, transposed=transposed)
        assert y.dtype == x.dtype and y.shape == (rows, outs)
        _check(y, x, w, transposed=transposed)
        assert torch.equal(store.linear(1, x, transposed=transposed), y)  # the same bits
        drop = (0.3, 99, 2)
        y = store.linear(1, x, bias=2, activation="gelu_tanh", dropout=drop, residual=res,
                         transposed=transposed)
        _check(y, x, w, b, "gelu_tanh", drop, res, transposed)
        # the input's gradient of a layer whose weight lies the other way round is the same product
        y = store.linear_input_grad(1, x, add=res, transposed=not transposed)
        _check(y, x, w, residual=res, transposed=transposed)


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("mode", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [3, 150])
def test_what_follows_the_product(activation, mode, rows):
    torch = torch_mod()
    x, w, b = _inputs(rows, 100, 70, mode, 7)
    with B.store_of([w, b], mode) as store:
        for dtype in (torch.float32, torch.bfloat16):
            res = (torch.arange(rows * 70, device="cuda").view(rows, 70) / 99).to(dtype)
            for bias in (None, 2):
                for drop in (None, (0.5, 3, 0)):
                    for r in (None, res):
                        y = store.linear(1, x, bias=bias, activation=activation, dropout=drop,
                                         residual=r, dtype=dtype)
                        assert y.dtype == dtype
                        _check(y, x, w, None if bias is None else b, activation, drop, r)


@pytest.mark.parametrize("mode", ["mixed", "fp32"])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows", [4, 140])
def test_strides_and_places(mode, transposed, rows):
    torch = torch_mod()
    for cols, outs in ((72, 136), (33, 50)):
        x, w, b = _inputs(rows, cols, outs, mode, 11, transposed)
        res = torch.randn(rows, outs, device="cuda").to(x.dtype)
        with B.store_of([w, b], mode) as store:
            want = store.linear(1, x, bias=2, residual=res, transposed=transposed)
            _check(want, x, w, b, residual=res, transposed=transposed)
            for left, right in ((1, 0), (8, 8), (3, 6)):
                xp = B.pitched(x, left, right, float("nan"))
                rp = B.pitched(res, right, left, float("nan"))
                out = B.pitched(torch.zeros_like(res), left, right, 7.0)
                got = store.linear(1, xp, bias=2, residual=rp, transposed=transposed, out=out)
                # (another path may take the sums in another order)
                assert got is out
                _check(got, x, w, b, residual=res, transposed=transposed)
                assert (out._base[:, :left] == 7).all()
                assert (out._base[:, left + outs:] == 7).all()
                store.linear(1, xp, bias=2, residual=rp, transposed=transposed, out=rp)
                assert torch.equal(rp, got)
            three = store.linear(1, x.view(2, rows // 2, cols), bias=2, transposed=transposed,
                                 residual=res.view(2, rows // 2, outs))
            assert torch.equal(three.view(rows, outs), want)
            one = store.linear(1, x[0], transposed=transposed)
            assert one.shape == (outs,)
            _check(one[None], x[:1], w, transposed=transposed)


# several tiles each way, long and short sums, sizes on and off every grid
LARGER = [(1025, 1600, 1601, "mixed"), (3000, 770, 523, "mixed"), (520, 6400, 1600, "mixed"),
          (2304, 1280, 1280, "bf16"), (700, 1284, 900, "fp32"), (4100, 64, 4100, "mixed"),
          (300, 50257, 100, "mixed"), (33, 768, 50257, "mixed"), (4099, 1288, 5128, "mixed"),
          (8200, 200, 1288, "bf16"), (8190, 2568, 1280, "mixed"), (5, 5128, 1288, "mixed"),
          (100, 5120, 1280, "mixed"), (1, 50264, 136, "mixed"), (17, 4001, 1201, "mixed"),
          (1, 768, 50257, "fp32"), (64, 6401, 300, "fp32"), (65, 6400, 301, "fp32"),
          (3, 40, 70001, "bf16")]


@pytest.mark.parametrize("rows,cols,outs,mode", LARGER)
@pytest.mark.parametrize("transposed", [False, True])
def test_larger_products(rows, cols, outs, mode, transposed):
    torch = torch_mod()
    x, w, b = _inputs(rows, cols, outs, mode, 13, transposed)
    res = torch.randn(rows, outs, device="cuda").to(x.dtype)
    with B.store_of([w, b], mode) as store:
        y = store.linear(1, x, bias=2, transposed=transposed)
        _check(y, x, w, b, transposed=transposed)
        y = store.linear(1, x, bias=2, activation="gelu", dropout=(0.1, 3, 1), residual=res,
                         transposed=transposed)
        _check(y, x, w, b, "gelu", (0.1, 3, 1), res, transposed)


@pytest.mark.parametrize("rows", [1, 9, 200])
@pytest.mark.parametrize("mode", ["mixed", "fp32"])
def test_infinities_and_nan(rows, mode):
    """An infinity in a row reaches that row's outputs as infinities (0 weights: NaN), a NaN as
    NaN; other rows do not change."""
    torch = torch_mod()
    x, w, _ = _inputs(rows, 90, 60, mode, 17)
    w[5, 3] = 0.0
    w[6] = 0.75  # (bf16 holds it: its second and third part are 0)
    with B.store_of([w], mode) as store:
        clean = store.linear(1, x)
        x[0, 5] = float("inf")
        y = store.linear(1, x)
        assert y[0, 3].isnan()
        assert torch.equal(y[0, 4:], torch.sign(w[5, 4:]).to(y.dtype) * float("inf"))
        assert torch.equal(y[1:], clean[1:])
        x[0, 5], x[0, 6] = 1.0, float("-inf")
        assert (store.linear(1, x)[0] == float("-inf")).all()
        x[0, 6] = float("nan")
        y = store.linear(1, x)
        assert y[0].isnan().all() and torch.equal(y[1:], clean[1:])
    x, w, _ = _inputs(rows, 90, 60, mode, 18)
    w[7, 11] = float("inf")
    with B.store_of([w], mode) as store:
        y = store.linear(1, x)
        assert torch.equal(y[:, 11], torch.sign(x[:, 7]) * float("inf"))
        assert y[:, :11].isfinite().all() and y[:, 12:].isfinite().all()


def test_exact_products():
    """Whole numbers whose sums fp32 holds come out exactly: every element is where it belongs."""
    torch = torch_mod()
    for mode in ("mixed", "fp32"):
        for rows, cols, outs in ((1, 40, 70), (7, 300, 33), (140, 130, 150), (300, 256, 520)):
            g = torch.Generator(device="cuda").manual_seed(rows)
            x = torch.randint(-8, 9, (rows, cols), generator=g, device="cuda").float()
            w = torch.randint(-8, 9, (cols, outs), generator=g, device="cuda").float()
            want = x.double() @ w.double()
            with B.store_of([w, w.t().contiguous()], mode) as store:
                xt = x.to(B.param_dtype(mode))
                for i, tr in ((1, False), (2, True)):
                    assert torch.equal(store.linear(i, xt, transposed=tr, dtype=torch.float32),
                                       want.float())


def test_full_precision_uses_all_bits():
    """fp32 operands whose lower bits decide: x is 1 + 2^-23, W's columns cancel its leading bits."""
    torch = torch_mod()
    for rows in (1, 160):
        x = torch.ones(rows, 64, device="cuda")
        x[:, 0] += 2.0 ** -23
        w = torch.zeros(64, 32, device="cuda")
        w[0], w[1] = 1.0, -1.0
        with B.store_of([w, torch.full((32,), 0.5, device="cuda")], "fp32") as store:
            assert (store.linear(1, x) == 2.0 ** -23).all()
            w2 = torch.zeros(64, 32, device="cuda")
        w2[0], w2[1] = 1.0 + 2.0 ** -20, -1.0
        with B.store_of([w2], "fp32") as store:  # (1 + 2^-20)(1 + 2^-23) - 1, to 2^-22 of it
            y = store.linear(1, x).double()
            assert ((y - (2.0 ** -20 + 2.0 ** -23 + 2.0 ** -43)).abs() <= 2.0 ** -22).all()


def test_captured_and_a_seed_on_the_device():
    torch = torch_mod()
    for rows in (1, 300):
        x, w, b = _inputs(rows, 256, 200, "mixed", 19)
        seed = torch.tensor([5], device="cuda")
        with B.store_of([w, b], "mixed") as store:
            store.set_stream(torch.cuda.Stream())
            torch.cuda.synchronize()
            y = store.linear(1, x, bias=2, activation="gelu", dropout=(0.2, seed, 1))
            dx = store.linear_input_grad(1, y, add=x)
            store.begin_capture()
            store.linear(1, x, bias=2, activation="gelu", dropout=(0.2, seed, 1), out=y)
            store.linear_input_grad(1, y, add=x, out=dx)
            graph = store.end_capture()
            for k in range(4):
                x.copy_(_inputs(rows, 256, 200, "mixed", 60 + k)[0])
                seed.fill_(k)
                torch.cuda.synchronize()
                graph.replay()
                store.sync()
                got = y.clone(), dx.clone()
                e = store.linear(1, x, bias=2, activation="gelu", dropout=(0.2, k, 1))
                d = store.linear_input_grad(1, e, add=x)
                torch.cuda.synchronize()
                assert torch.equal(got[0], e) and torch.equal(got[1], d)
            graph.close()


def test_two_stores_on_two_streams_at_once():
    torch = torch_mod()
    sets = []
    for k in range(2):
        x, w, b = _inputs(5 + 300 * k, 512, 640, "mixed", 23 + k)
        store = B.store_of([w, b], "mixed")
        store.set_stream(torch.cuda.Stream())
        torch.cuda.synchronize()
        sets.append((store, x, w, b, []))
    for _ in range(5):
        for store, x, w, b, got in sets:
            got.append(store.linear(1, x, bias=2))
    torch.cuda.synchronize()
    for store, x, w, b, got in sets:
        _check(got[0], x, w, b)
        assert all(torch.equal(g, got[0]) for g in got)
        store.close()


def test_rows_past_32_bits_of_elements():
    """Rows of x and y 2^31 elements apart: the last begins past 2^32."""
    torch = torch_mod()
    pitch = 2 ** 31
    x, w, b = _inputs(3, 64, 48, "mixed", 29)
    far = torch.empty(2 * pitch + 64, dtype=torch.bfloat16, device="cuda")
    xf = far.as_strided((3, 64), (pitch, 1))
    xf.copy_(x)
    of = torch.empty(2 * pitch + 64, dtype=torch.bfloat16, device="cuda").as_strided(
        (3, 48), (pitch, 1))
    with B.store_of([w, b], "mixed") as store:
        store.linear(1, xf, bias=2, out=of)
        _check(of, x, w, b)


def test_refusals():
    import ttperf
    torch = torch_mod()
    x, w, b = _inputs(6, 16, 24, "mixed", 31)
    with B.store_of([w, b], "mixed") as store:
        out = torch.zeros(6, 24, dtype=torch.bfloat16, device="cuda")
        for bad in (dict(index=0), dict(index=2), dict(index=9), dict(index=-1), dict(index=None),
                    dict(bias=3), dict(bias=-1), dict(bias=1), dict(transposed=True),
                    dict(x=x.float()), dict(x=x.cpu()), dict(x=x[:, :15]), dict(x=x.t()),
                    dict(activation="swish"), dict(dropout=(1.0, 1, 0)), dict(dropout=(0.1, 1, -1)),
                    dict(residual=out[:5]), dict(residual=out.float()), dict(dtype=torch.float16),
                    dict(out=out[:, :23]), dict(out=out.float(), dtype=torch.bfloat16),
                    dict(residual=out, dtype=torch.float32)):
            a = dict(dict(index=1, x=x), **bad)
            with pytest.raises((ValueError, ttperf.TTPError)):
                store.linear(a.pop("index"), a.pop("x"), **a)
        with pytest.raises(ValueError):
            store.linear_input_grad(1, x)  # 16 columns; the outputs are 24
        flat = torch.zeros(6 * 24 + 6 * 16, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(ValueError, match="overlap"):
            store.linear(1, flat[:96].view(6, 16), out=flat[90:90 + 144].view(6, 24))
        with pytest.raises(ValueError, match="overlap"):
            store.linear(1, x, residual=flat[:144].view(6, 24), out=flat[1:145].view(6, 24))
        weight = store.tensors[1].torch_view().view(-1)
        with pytest.raises(ValueError, match="overlap"):
            store.linear(1, x, out=weight[:144].view(6, 24))
        assert (out == 0).all() and (flat == 0).all()
        assert store.linear(1, x[:0]).shape == (0, 24)
