"""GPU tests of a linear layer's gradients from its input kept in 8 bits, into the store, against
products in 64 bits.

Tolerances: the kept values are exact in bf16 and an fp32 dy is the sum of its three bf16 parts, so
the products are exact; sums are fp32 chains of N / 16 matrix instructions of 16 products and the
parts' additions, each a rounding: (N / 16 + 64) u of the sum of magnitudes, u = 2^-24.  The bias
sums chains of at most N / 8 + 64.  Then one rounding to the gradient's type: 2^-8 in bf16."""
import math

import pytest

from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _store(cols, outs, mode="mixed", transposed=False):
    import ttperf
    torch = torch_mod()
    # a tensor on either side: nothing else of the gradients may change
    w = (outs, cols) if transposed else (cols, outs)
    s = ttperf.ParamStore([(100,), w, (outs,), (70,)], mode=mode)
    s.set_stream(torch.cuda.current_stream())
    return s


def _inputs(rows, cols, outs, dtype, seed, pitch=0):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g, device="cuda").float())
    wide = torch.randn(rows, outs + pitch, generator=g, device="cuda").to(dtype)
    return x, wide[:, pitch // 2:pitch // 2 + outs]


def _check(store, kept, dy, transposed, old=None, bias=True):
    import ttperf
    torch = torch_mod()
    x = store.restore8(kept, dtype=torch.float32).double().cpu()
    d = dy.double().cpu()
    rows = x.shape[0]
    dw = store.tensors[1].torch_view(ttperf.BUF_GRAD)
    unit = 2.0 ** -8 if dw.dtype == torch.bfloat16 else U
    for got, want, mag, chain, before in (
            (dw, x.t() @ d, x.abs().t() @ d.abs(), rows / 16 + 64, old and old[0]),
            (store.tensors[2].torch_view(ttperf.BUF_GRAD), d.sum(0), d.abs().sum(0),
             rows / 8 + 64, old and old[1])):
        if want.dim() == 1 and not bias:
            continue
        if want.dim() == 2 and transposed:
            want, mag = want.t(), mag.t()
        if old:
            want = want + before.double().cpu()
        tol = chain * U * mag + unit * want.abs() + U * want.abs()
        err = (got.double().cpu() - want).abs()
        assert (err <= tol).all(), float((err / tol.clamp(min=1e-300)).max())


SHAPES = [(1, 1, 1), (1, 40, 33), (5, 32, 8), (31, 33, 7), (32, 128, 128), (33, 129, 130),
          (100, 65, 257), (257, 384, 160), (300, 31, 1000), (1000, 200, 64), (4099, 96, 72)]


@pytest.mark.parametrize("rows,cols,outs", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("transposed", [False, True])
def test_gradients(rows, cols, outs, dtype, fmt, transposed):
    import ttperf
    torch = torch_mod()
    x, dy = _inputs(rows, cols, outs, getattr(torch, dtype), rows + cols + outs)
    mode = "fp32" if dtype == "float32" else "mixed"
    with _store(cols, outs, mode, transposed) as store:
        kept = store.checkpoint8(x, fmt=fmt)
        flat = store.torch_view(ttperf.BUF_GRAD)
        flat.fill_(3.0)
        before = flat.clone()
        store.accumulate_linear_grad8(1, kept, dy, bias=2, transposed=transposed)
        assert [store.has_grad(i) for i in range(4)] == [False, True, True, False]
        _check(store, kept, dy, transposed)
        # nothing else of the buffer was written, the padding among it
        mask = torch.ones(store.total, dtype=torch.bool, device="cuda")
        for i in (1, 2):
            mask[store.offsets[i]:store.offsets[i] + store.tensors[i].numel] = False
        assert torch.equal(flat[mask], before[mask])
        # a second micro-batch is added; the same inputs give the same bits
        first = [store.tensors[i].torch_view(ttperf.BUF_GRAD).clone() for i in (1, 2)]
        store.accumulate_linear_grad8(1, kept, dy, bias=2, transposed=transposed)
        _check(store, kept, dy, transposed, old=first)
        store.zero_grad()
        store.accumulate_linear_grad8(1, kept, dy, bias=2, transposed=transposed)
        for i, f in zip((1, 2), first):
            assert torch.equal(store.tensors[i].torch_view(ttperf.BUF_GRAD), f)


@pytest.mark.parametrize("mode,dtype", [("mixed", "float32"), ("fp32", "bfloat16"),
                                        ("bf16", "bfloat16")])
def test_a_gradient_of_another_type_than_the_stores(mode, dtype):
    torch = torch_mod()
    for rows, cols, outs in ((70, 50, 33), (2000, 130, 96)):
        x, dy = _inputs(rows, cols, outs, getattr(torch, dtype), 9, pitch=7)
        with _store(cols, outs, mode) as store:
            kept = store.checkpoint8(x)
            store.accumulate_linear_grad8(1, kept, dy, bias=2)
            _check(store, kept, dy, False)


def test_larger_tiles_and_strides():
    """Sizes with several tiles each way and none, several or many parts; rows of dy at an odd
    pitch and offset."""
    torch = torch_mod()
    for rows, cols, outs, dtype, fmt, transposed in (
            (512, 2100, 2050, torch.bfloat16, "int8", False),
            (700, 2100, 1030, torch.float32, "int8", True),
            (9000, 300, 500, torch.bfloat16, "e4m3", True),
            (3585, 384, 1536, torch.float32, "int8", False),
            (16384, 64, 65, torch.float32, "e4m3", False)):
        x, dy = _inputs(rows, cols, outs, dtype, rows, pitch=3)
        with _store(cols, outs, "mixed" if dtype == torch.bfloat16 else "fp32",
                    transposed) as store:
            kept = store.checkpoint8(x, fmt=fmt)
            store.accumulate_linear_grad8(1, kept, dy, bias=2, transposed=transposed)
            _check(store, kept, dy, transposed)
            only = [store.tensors[i].grad.numpy() for i in (1, 2)]
            store.zero_grad()
            store.accumulate_linear_grad8(1, kept, dy, transposed=transposed)  # no bias
            assert (store.tensors[1].grad.numpy() == only[0]).all()
            assert not store.has_grad(2)


def test_no_rows():
    """No tokens: a first gradient is zero, a further one leaves it."""
    import ttperf
    torch = torch_mod()
    x, dy = torch.empty(0, 40, device="cuda"), torch.empty(0, 24, device="cuda")
    with _store(40, 24) as store:
        kept = store.checkpoint8(x)
        store.torch_view(ttperf.BUF_GRAD).fill_(5.0)
        store.accumulate_linear_grad8(1, kept, dy, bias=2)
        assert (store.tensors[1].grad.numpy() == 0).all()
        assert (store.tensors[2].grad.numpy() == 0).all()
        store.torch_view(ttperf.BUF_GRAD).fill_(5.0)
        store.accumulate_linear_grad8(1, kept, dy, bias=2)
        assert (store.tensors[1].grad.numpy() == 5).all()


def test_what_is_not_finite_reaches_the_gradient():
    """An infinity in the activation (its block stands for NaN) or in dy: NaN or infinity in every
    gradient that it touches, and nowhere else."""
    torch = torch_mod()
    for dtype in (torch.bfloat16, torch.float32):
        for fmt in ("int8", "e4m3"):
            x, dy = _inputs(90, 100, 70, dtype, 4)
            x[17, 40] = math.inf
            dy[60, 9] = math.nan
            with _store(100, 70, "mixed" if dtype == torch.bfloat16 else "fp32") as store:
                kept = store.checkpoint8(x, fmt=fmt)
                store.accumulate_linear_grad8(1, kept, dy, bias=2)
                dw = torch.from_numpy(store.tensors[1].grad.numpy())
                db = torch.from_numpy(store.tensors[2].grad.numpy())
            bad = torch.zeros(100, 70, dtype=torch.bool)
            bad[32:64] = True
            bad[:, 9] = True
            assert torch.equal(~dw.isfinite(), bad)
            assert (~db.isfinite()).nonzero().flatten().tolist() == [9]


def test_the_largest_numbers():
    """dy up to the type's largest: its parts stay finite (the gradients too, under a small x)."""
    torch = torch_mod()
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.full((40, 32), 2.0 ** -20, device="cuda")
        dy = torch.full((40, 24), torch.finfo(dtype).max, device="cuda", dtype=dtype)
        dy[::2] = -dy[::2] / 2
        with _store(32, 24, "fp32") as store:
            kept = store.checkpoint8(x)
            store.accumulate_linear_grad8(1, kept, dy)
            _check(store, kept, dy, False, bias=False)


def test_against_differences():
    """The gradient of sum(dy * (x W + b)) in W and b by differences: it is linear, so a difference
    over a step of 1 is exact but for the rounding of the loss."""
    torch = torch_mod()
    x, dy = _inputs(20, 35, 9, torch.float32, 2)
    with _store(35, 9, "fp32") as store:
        kept = store.checkpoint8(x)
        xk = store.restore8(kept).double().cpu()
        store.accumulate_linear_grad8(1, kept, dy, bias=2)
        dw, db = (store.tensors[i].grad.numpy() for i in (1, 2))
    d = dy.double().cpu()
    w = torch.randn(35, 9, dtype=torch.float64)
    b = torch.randn(9, dtype=torch.float64)

    def loss(w, b):
        return float((d * (xk @ w + b)).sum())
    base, mag = loss(w, b), float((xk.abs().t() @ d.abs()).max())
    for i, o in ((0, 0), (34, 8), (17, 3), (31, 5), (32, 5)):
        up = w.clone()
        up[i, o] += 1
        assert abs(loss(up, b) - base - dw[i, o]) <= 80 * U * mag + 1e-11 * abs(base)
        ub = b.clone()
        ub[o] += 1
        assert abs(loss(w, ub) - base - db[o]) <= 80 * U * mag + 1e-11 * abs(base)


def test_the_step_takes_it():
    """A gradient made this way and the same one accumulated: bit-equal steps, norms and sums; a
    gradient sum taken before it is stale."""
    import ttperf
    torch = torch_mod()
    x, dy = _inputs(300, 96, 80, torch.bfloat16, 1)
    with _store(96, 80) as a, _store(96, 80) as b:
        for s in (a, b):
            s.configure_scaler(True, init_scale=8.0)
            for t in s.tensors:
                t.set_data(torch.linspace(-1, 1, t.numel).numpy())
        kept = a.checkpoint8(x)
        a.accumulate_linear_grad8(1, kept, dy, bias=2)
        b.accumulate_grads([1, 2], [a.tensors[i].torch_view(ttperf.BUF_GRAD).clone()
                                    for i in (1, 2)])
        assert a.grad_norm() == b.grad_norm()
        ra, rb = (s.adam_step(1e-2, max_grad_norm=1.0, report=True) for s in (a, b))
        assert ra == rb
        for i in (1, 2):
            assert (a.tensors[i].numpy() == b.tensors[i].numpy()).all()
        a.grad_sumsq_tensors([1, 2])
        a.accumulate_linear_grad8(1, kept, dy, bias=2)
        with pytest.raises(ttperf.TTPError):
            a.adam_step(1e-2, max_grad_norm=1.0, tensor_sums=True, indices=[1, 2])


def test_captured():
    """In a captured backward: assigns at every replay, with other inputs."""
    import ttperf
    torch = torch_mod()
    s = torch.cuda.Stream()
    for rows, cols, outs in ((64, 40, 24), (3000, 130, 96)):
        store = ttperf.ParamStore([(cols, outs), (outs,)], mode="mixed")
        store.set_stream(s)
        with torch.cuda.stream(s):
            x, dy = _inputs(rows, cols, outs, torch.bfloat16, 3)
            dy = dy.contiguous()
            kept = store.checkpoint8(x)
            store.accumulate_linear_grad8(0, kept, dy, bias=1)
            store.sync()
            store.begin_capture()
            with pytest.raises(ttperf.TTPError):  # its first write has to follow a zero_grad
                store.accumulate_linear_grad8(0, kept, dy, bias=1)
            store.zero_grad(fill=False)
            store.checkpoint8(x, out=kept)
            store.accumulate_linear_grad8(0, kept, dy, bias=1)
            graph = store.end_capture()
            for k in range(4):
                x.copy_(torch.randn(rows, cols, device="cuda"))
                dy.copy_(torch.randn(rows, outs, device="cuda"))
                graph.replay()
                torch.cuda.synchronize()
                got = [store.tensors[i].torch_view(ttperf.BUF_GRAD).clone() for i in (0, 1)]
                store.zero_grad()
                store.accumulate_linear_grad8(0, store.checkpoint8(x), dy, bias=1)
                for i in (0, 1):
                    assert torch.equal(got[i], store.tensors[i].torch_view(ttperf.BUF_GRAD))
        graph.close()
        store.close()


def test_refusals():
    import ttperf
    torch = torch_mod()
    x, dy = _inputs(20, 40, 24, torch.bfloat16, 5)
    with _store(40, 24) as store:
        kept = store.checkpoint8(x)

        def refused(call, exc=ValueError):
            with pytest.raises(exc):
                call()
            assert not any(store.has_grad(i) for i in range(4))
        refused(lambda: store.accumulate_linear_grad8(1, x, dy))
        refused(lambda: store.accumulate_linear_grad8(9, kept, dy))
        refused(lambda: store.accumulate_linear_grad8(1, kept, dy, bias=9))
        refused(lambda: store.accumulate_linear_grad8(1, kept, dy, bias=1))
        refused(lambda: store.accumulate_linear_grad8(0, kept, dy))
        refused(lambda: store.accumulate_linear_grad8(1, kept, dy, bias=3))
        refused(lambda: store.accumulate_linear_grad8(1, kept, dy[:19]))
        refused(lambda: store.accumulate_linear_grad8(1, kept, dy[:, :23]))
        refused(lambda: store.accumulate_linear_grad8(1, kept, dy.half()))
        refused(lambda: store.accumulate_linear_grad8(1, kept, dy.cpu()))
        # dy in the store's own gradients
        own = store.torch_view(ttperf.BUF_GRAD)[:480].view(20, 24)
        refused(lambda: store.accumulate_linear_grad8(1, kept, own))
