"""GPU tests of dropout: every element equals the formula's, with the generator on the host.  The
factor's product and the sum with the residual are one fp32 rounding each, then one to the type, on
either side: the results have the same bits."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu


@pytest.fixture
def store():
    s = B.store_of([], "fp32")
    yield s
    s.close()


def _x(rows, cols, dtype, seed):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, cols, generator=g, device="cuda").to(dtype)


def _want(x, p, seed, stream, residual=None):
    r = None if residual is None else residual.float().cpu()
    return B.dropped(x.float().cpu(), p, seed, stream, r).to(x.dtype)


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 9), (1, 4097), (33, 384), (257, 65), (1021, 130), (4099, 16)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("residual", [False, True])
def test_elements(store, rows, cols, dtype, residual):
    torch = torch_mod()
    dtype = getattr(torch, dtype)
    x = _x(rows, cols, dtype, 1)
    r = _x(rows, cols, dtype, 2) if residual else None
    for p, seed, stream in ((0.1, 12345, 0), (0.5, 2 ** 64 - 3, 2 ** 40 + 9), (0.999, -7, 1)):
        y = store.dropout(x, p, seed, stream=stream, residual=r)
        assert torch.equal(y.cpu(), _want(x, p, seed, stream, r)), (p, seed, stream)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_strides_offsets_and_places(store, dtype):
    torch = torch_mod()
    dtype = getattr(torch, dtype)
    for cols, left, right in ((50, 1, 4), (64, 3, 0), (129, 8, 8)):
        x, r = _x(40, cols, dtype, 3), _x(40, cols, dtype, 4)
        want = _want(x, 0.3, 99, 5, r)
        xp, rp = B.pitched(x, left, right), B.pitched(r, right, left)
        out = B.pitched(torch.zeros_like(x), left, right, 7.0)
        assert store.dropout(xp, 0.3, 99, stream=5, residual=rp, out=out) is out
        assert torch.equal(out.cpu(), want)
        whole = out._base
        assert (whole[:, :left] == 7).all() and (whole[:, left + cols:] == 7).all()
        a = xp.clone()
        store.dropout(a, 0.3, 99, stream=5, residual=r, out=a)  # in the input's place
        assert torch.equal(a.cpu(), want)
        store.dropout(xp, 0.3, 99, stream=5, residual=rp, out=rp)  # in the residual's
        assert torch.equal(rp.cpu(), want)
        same = xp.clone()  # the input is the residual, too
        store.dropout(same, 0.3, 99, residual=same, out=same)
        assert torch.equal(same.cpu(), _want(x, 0.3, 99, 0, x))


def test_the_rows_of_more_dimensions(store):
    torch = torch_mod()
    x = _x(12, 20, torch.float32, 5)
    y = store.dropout(x.view(3, 4, 20), 0.2, 1)
    assert y.shape == (3, 4, 20) and torch.equal(y.view(12, 20).cpu(), _want(x, 0.2, 1, 0))
    assert torch.equal(store.dropout(x[0], 0.2, 1).cpu(), _want(x[:1], 0.2, 1, 0)[0])


def test_dropped_elements_are_zero_or_the_residual_whatever_they_were(store):
    torch = torch_mod()
    keep = torch.from_numpy(B.kept(64, 33, 0.5, 3, 0))
    x = torch.full((64, 33), float("inf"), device="cuda")
    x[::2] = float("nan")
    y = store.dropout(x, 0.5, 3).cpu()
    assert (y[~keep] == 0).all()
    assert (y[1::2][keep[1::2]] == float("inf")).all() and y[::2][keep[::2]].isnan().all()
    r = _x(64, 33, torch.float32, 6)
    y = store.dropout(x, 0.5, 3, residual=r).cpu()
    assert torch.equal(y[~keep], r.cpu()[~keep])


def test_p_zero_keeps_all_and_the_share_is_p(store):
    torch = torch_mod()
    x = _x(77, 51, torch.bfloat16, 7)
    assert torch.equal(store.dropout(x, 0.0, 1), x)
    ones = torch.ones(2048, 1024, device="cuda")
    for p in (0.1, 0.37):
        y = store.dropout(ones, p, 11)
        n = ones.numel()
        share = float((y == 0).sum()) / n
        assert abs(share - p) < 6 * (p * (1 - p) / n) ** 0.5 + 2.0 ** -17
        # rows, columns and places within a group do not stand out (6 deviations of 1024 or more)
        for dim, m in ((0, 2048), (1, 1024)):
            part = (y == 0).float().mean(dim)
            assert float((part - p).abs().max()) < 6 * (p * (1 - p) / m) ** 0.5
    # other seeds and streams: other masks
    a, b, c = store.dropout(ones, 0.5, 1), store.dropout(ones, 0.5, 2), \
        store.dropout(ones, 0.5, 1, stream=1)
    for u, v in ((a, b), (a, c), (b, c)):
        assert abs(float((u == v).float().mean()) - 0.5) < 0.003


def test_the_gradient_is_the_same_call(store):
    """dropout(dy) with the forward's numbers is the derivative of sum(dy y) by x: y is linear in x,
    so the difference for one element moved by 1 is the factor or 0."""
    torch = torch_mod()
    x, dy = _x(9, 21, torch.float32, 8), torch.ones(9, 21, device="cuda")
    g = store.dropout(dy, 0.4, 77, stream=3)
    y0 = store.dropout(x, 0.4, 77, stream=3).double()
    y1 = store.dropout(x + 1, 0.4, 77, stream=3).double()
    # fp32 roundings of values up to 8 on both sides: x + 1, two products
    assert (((y1 - y0) - g.double()).abs() <= 3 * 8 * 2 * B.U).all()


def test_a_seed_on_the_device_and_captured_calls():
    torch = torch_mod()
    seed = torch.tensor([41], device="cuda")
    x = _x(100, 70, torch.bfloat16, 9)
    with B.store_of([], "fp32") as store:
        assert torch.equal(store.dropout(x, 0.2, seed).cpu(), _want(x, 0.2, 41, 0))
        side = torch.cuda.Stream()
        store.set_stream(side)
        out, out2 = torch.empty_like(x), torch.empty_like(x)
        torch.cuda.synchronize()
        with pytest.raises(ValueError):
            store.begin_capture()
            try:
                store.dropout(x, 0.2, seed)  # a result has to be given
            finally:
                store.end_capture(discard=True)
        store.begin_capture()
        store.dropout(x, 0.2, seed, out=out)
        store.dropout(out, 0.2, 5, stream=1, residual=x, out=out2)
        graph = store.end_capture()
        for k in range(4):
            seed.fill_(k * 1000 - 1)
            torch.cuda.synchronize()
            graph.replay()
            store.sync()
            assert torch.equal(out.cpu(), _want(x, 0.2, k * 1000 - 1, 0))
            assert torch.equal(out2.cpu(), _want(out, 0.2, 5, 1, x))
            torch.randn(1000, device="cuda").sum().item()  # other work between the launches
        graph.close()


def test_a_store_on_a_stream_of_its_own():
    import ttperf
    torch = torch_mod()
    store = ttperf.ParamStore([(64,)])
    for k in range(3):
        x = _x(2000, 500, torch.float32, 20 + k)
        y = store.dropout(x, 0.1, k)
        want = _want(x, 0.1, k, 0)
        del x
        torch.empty(2000, 500, device="cuda").fill_(9)  # the memory may be given out again
        assert torch.equal(y.cpu(), want)
    store.close()


def test_offsets_past_32_bits(store):
    """Rows 2^31 elements apart: the third begins past 2^32."""
    torch = torch_mod()
    pitch, cols = 2 ** 31, 40
    x = torch.empty(2 * pitch + cols, dtype=torch.bfloat16, device="cuda").as_strided(
        (3, cols), (pitch, 1))
    x.copy_(_x(3, cols, torch.bfloat16, 10))
    want = _want(x, 0.25, 6, 0)
    store.dropout(x, 0.25, 6, out=x)
    assert torch.equal(x.cpu(), want)


def test_refusals(store):
    torch = torch_mod()
    x = _x(8, 16, torch.float32, 11)
    before = x.clone()
    for bad in (dict(p=1.0), dict(p=-0.1), dict(p=float("nan")), dict(seed=2 ** 64),
                dict(stream=-1), dict(stream=2 ** 64), dict(seed=torch.tensor([1])),
                dict(seed=torch.tensor([1, 2], device="cuda")),
                dict(residual=x[:4]), dict(residual=x.bfloat16()), dict(out=x.bfloat16()),
                dict(out=torch.empty(8, 17, device="cuda")), dict(x=x.half()), dict(x=x.cpu()),
                dict(x=x.t()), dict(x=torch.empty(3, 0, device="cuda"))):
        args = dict(dict(x=x, p=0.5, seed=1), **bad)
        with pytest.raises(ValueError):
            store.dropout(args.pop("x"), args.pop("p"), args.pop("seed"), **args)
    flat = torch.zeros(8 * 16 + 8, device="cuda")
    a, b = flat[:128].view(8, 16), flat[8:].view(8, 16)
    with pytest.raises(ValueError, match="overlap"):
        store.dropout(a, 0.5, 1, out=b)
    with pytest.raises(ValueError, match="overlap"):
        store.dropout(x, 0.5, 1, residual=a, out=b)
    with pytest.raises(ValueError, match="overlap"):  # the seed in the result
        store.dropout(x, 0.5, flat.view(torch.int64)[:1], out=a)
    assert torch.equal(x, before) and (flat == 0).all()
    assert store.dropout(torch.empty(0, 5, device="cuda"), 0.5, 1).shape == (0, 5)
