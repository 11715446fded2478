"""GPU tests of the embedding lookup and its gradient.

The lookup rounds as its formula does (scale times the entry, plus the position's, then to the type):
the same bits.  The gradient's row is a chain of at most 32 fp32 additions in each of n / 32 + 2 parts
and one over the parts: (34 + n / 32) u of the sum of magnitudes, u = 2^-24, then one product, at most
one addition and one rounding."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
U = B.U


def _table(vocab, cols, mode, seed=0):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(vocab, cols, generator=g, device="cuda").to(B.param_dtype(mode)).float()


def _tokens(rows, vocab, seed, kind="zipf"):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "same":
        t = torch.full((rows,), vocab // 2, device="cuda")
    elif kind == "positions":
        t = torch.arange(rows, device="cuda") % vocab
    elif kind == "uniform":
        t = torch.randint(vocab, (rows,), generator=g, device="cuda")
    else:
        u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        t = (torch.exp(u * torch.log(torch.tensor(vocab + 1.0))) - 1).long().clamp(0, vocab - 1)
        hide = torch.rand(rows, generator=g, device="cuda")
        t[hide < 0.05] = -1
        t[hide > 0.97] = vocab + 3
    return t


def _looked_up(w, t, scale, dtype):
    """The formula in fp32, a rounding each."""
    torch = torch_mod()
    rows = w[t.clamp(0, w.shape[0] - 1)]
    rows = torch.where((t < 0)[:, None], 0.0, rows)
    return torch.where((t >= w.shape[0])[:, None], float("nan"), rows) * scale


SHAPES = [(1, 1, 1), (1, 768, 1000), (3, 7, 2), (65, 384, 65), (257, 33, 1025), (1000, 260, 50257),
          (5, 4099, 3), (2050, 64, 9)]


@pytest.mark.parametrize("rows,cols,vocab", SHAPES)
@pytest.mark.parametrize("mode,dtype", [("mixed", "bfloat16"), ("fp32", "float32"),
                                        ("bf16", "float32"), ("fp32", "bfloat16")])
def test_lookup(rows, cols, vocab, mode, dtype):
    torch = torch_mod()
    dtype = getattr(torch, dtype)
    w, p = _table(vocab, cols, mode), _table(17, cols, mode, 1)
    t = _tokens(rows, vocab, rows)
    at = _tokens(rows, 17, rows + 1, "uniform")
    at[::5] = -2
    with B.store_of([w, p], mode) as store:
        for scale in (1.0, float(torch.tensor(cols).sqrt())):
            s = torch.tensor(scale, device="cuda")
            y = store.embedding(1, t, scale=scale, dtype=dtype)
            assert y.shape == (rows, cols) and y.dtype == dtype
            want = _looked_up(w, t, s, dtype)
            assert torch.equal(y.isnan(), want.isnan())
            assert torch.equal(y.nan_to_num(), want.to(dtype).nan_to_num())
            y = store.embedding(1, t, scale=scale, position=2, positions=at, dtype=dtype)
            want = want + _looked_up(p, at, 1.0, dtype)
            assert torch.equal(y.nan_to_num(), want.to(dtype).nan_to_num())
        assert store.embedding(1, t).dtype == B.param_dtype(mode)


def test_lookup_of_shapes_and_into_pitched_rows():
    torch = torch_mod()
    w = _table(50, 37, "mixed")
    with B.store_of([w], "mixed") as store:
        t = _tokens(24, 50, 1, "uniform")
        want = w[t].bfloat16()
        assert torch.equal(store.embedding(1, t.view(2, 3, 4)).view(24, 37), want)
        assert torch.equal(store.embedding(1, t.view(4, 6).t()).view(24, 37),
                           w[t.view(4, 6).t().reshape(-1)].bfloat16())
        assert torch.equal(store.embedding(1, t[3]), want[3])
        for left, right in ((1, 0), (5, 6)):
            out = B.pitched(torch.zeros_like(want), left, right, 7.0)
            assert store.embedding(1, t, out=out) is out
            assert torch.equal(out, want)
            assert (out._base[:, :left] == 7).all() and (out._base[:, left + 37:] == 7).all()
        assert store.embedding(1, t[:0]).shape == (0, 37)


def _check_grad(store, w, tokens, dys, scale, firsts=None):
    """The table's gradient after micro-batches of (tokens, dy)."""
    torch = torch_mod()
    got = B.grad(store, 1).double()
    vocab, cols = w.shape
    want = torch.zeros(vocab, cols, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    step = B.unit(B.grad(store, 1).dtype)
    for t, dy in zip(tokens, dys):
        live = (t >= 0) & (t < vocab)
        n = torch.zeros(vocab, dtype=torch.float64, device="cuda")
        n.index_add_(0, t[live], torch.ones_like(t[live], dtype=torch.float64))
        d = dy.double()[live] * scale
        mag = torch.zeros_like(want).index_add_(0, t[live], d.abs())
        want.index_add_(0, t[live], d)
        # additions that a term goes through: 16 in a chunk, then every fourth chunk's sum, and 4; up
        # to 512 rows every eighth term, and 4
        depth = torch.maximum(36 + n / 32, 4 + n / 8) if t.numel() <= 512 else 36 + n / 32
        tol += depth[:, None] * U * mag
        tol += (step + 2 * U) * (want.abs() + tol)
    err = (got - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-300)).max())


GRADS = [(1, 1, 1, "same"), (1, 768, 300, "uniform"), (31, 8, 5, "zipf"), (32, 130, 2, "same"),
         (33, 64, 3, "same"), (64, 257, 1000, "zipf"), (100, 33, 65, "uniform"),
         (1025, 384, 65, "zipf"), (4099, 48, 50257, "zipf"), (3000, 20, 3000, "positions"),
         (2048, 100, 128, "positions"), (5000, 36, 700, "same"), (2500, 768, 300, "zipf"),
         (700, 5, 20000, "uniform"), (20011, 8, 65, "zipf"), (40001, 12, 900, "zipf"),
         (512, 300, 3000, "zipf"), (513, 300, 3000, "zipf"), (512, 40, 9, "same"),
         (300, 40, 40001, "zipf"), (200, 257, 50257, "positions"), (100, 3, 40000, "uniform"),
         (1000, 3, 50, "zipf"), (600, 2, 5, "same")]


@pytest.mark.parametrize("rows,cols,vocab,kind", GRADS)
@pytest.mark.parametrize("mode,dtype", [("mixed", "bfloat16"), ("fp32", "float32"),
                                        ("bf16", "float32"), ("fp32", "bfloat16")])
def test_gradient(rows, cols, vocab, kind, mode, dtype):
    import ttperf
    torch = torch_mod()
    dtype = getattr(torch, dtype)
    w = torch.zeros(vocab, cols, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(rows)
    t = [_tokens(rows, vocab, rows + k, kind) for k in range(2)]
    dy = [torch.randn(rows, cols, generator=g, device="cuda").to(dtype) for _ in range(2)]
    with B.store_of([w], mode) as store:
        store.torch_view(ttperf.BUF_GRAD).fill_(3.0)
        store.accumulate_embedding_grad(1, t[0], dy[0], scale=1.5)
        assert [store.has_grad(i) for i in range(3)] == [False, True, False]
        _check_grad(store, w, t[:1], dy[:1], 1.5)
        assert B.untouched(store, (1,), 3.0)
        first = B.grad(store, 1).clone()
        store.accumulate_embedding_grad(1, t[1], dy[1], scale=1.5)
        _check_grad(store, w, t, dy, 1.5)
        # rows that the second one does not name are as they were
        named = torch.zeros(vocab, dtype=torch.bool, device="cuda")
        named[t[1][(t[1] >= 0) & (t[1] < vocab)]] = True
        assert torch.equal(B.grad(store, 1)[~named], first[~named])
        store.zero_grad()
        store.accumulate_embedding_grad(1, t[0], dy[0], scale=1.5)
        assert torch.equal(B.grad(store, 1), first)  # the same bits


def test_a_rows_sum_depends_on_its_tokens_alone():
    """The order of the additions is the rows' own: other tokens among them change nothing where the
    run lies in one chunk, and one row comes out exactly."""
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(1)
    with B.store_of([torch.zeros(900, 40, device="cuda")], "fp32") as store:
        t = torch.randperm(900, generator=g, device="cuda")
        dy = torch.randn(900, 40, generator=g, device="cuda")
        store.accumulate_embedding_grad(1, t, dy)
        assert torch.equal(B.grad(store, 1)[t], dy)


@pytest.mark.parametrize("rows", [60, 720])
def test_gradient_of_strided_rows_and_shapes(rows):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.zeros(30, 70, device="cuda")
    with B.store_of([w], "mixed") as store:
        t = _tokens(rows, 30, 5)
        dy = torch.randn(rows, 70, generator=g, device="cuda").bfloat16()
        store.accumulate_embedding_grad(1, t, dy)
        want = B.grad(store, 1).clone()
        for left, right in ((1, 2), (3, 8)):
            store.zero_grad()
            store.accumulate_embedding_grad(1, t, B.pitched(dy, left, right, float("nan")))
            assert torch.equal(B.grad(store, 1), want)
        store.zero_grad()
        store.accumulate_embedding_grad(1, t.view(4, -1), dy.view(4, -1, 70))
        assert torch.equal(B.grad(store, 1), want)


def test_no_rows_and_nothing_but_padding():
    import ttperf
    torch = torch_mod()
    with B.store_of([torch.zeros(30, 20, device="cuda")], "mixed") as store:
        store.torch_view(ttperf.BUF_GRAD).fill_(2.0)
        none = torch.empty(0, dtype=torch.int64, device="cuda")
        store.accumulate_embedding_grad(1, none, torch.empty(0, 20, device="cuda"))
        assert (B.grad(store, 1) == 0).all() and store.has_grad(1)
        B.grad(store, 1).fill_(2.0)
        pad = torch.full((100,), -1, device="cuda")
        nan = torch.full((100, 20), float("nan"), device="cuda")
        store.accumulate_embedding_grad(1, pad, nan)
        assert (B.grad(store, 1) == 2).all()
        store.zero_grad()
        store.accumulate_embedding_grad(1, pad, nan)
        assert (B.grad(store, 1) == 0).all() and B.untouched(store, (1,), 0.0)


@pytest.mark.parametrize("rows", [80, 800])
def test_infinities_and_nan_stay_in_their_rows(rows):
    torch = torch_mod()
    with B.store_of([torch.zeros(40, 12, device="cuda")], "fp32") as store:
        t = torch.arange(rows, device="cuda") % 40
        dy = torch.ones(rows, 12, device="cuda")
        dy[3], dy[4, 5] = float("inf"), float("nan")
        store.accumulate_embedding_grad(1, t, dy)
        g = B.grad(store, 1)
        assert (g[3] == float("inf")).all() and g[4, 5].isnan()
        g[3], g[4, 5] = rows // 40, rows // 40
        assert (g == rows // 40).all()


@pytest.mark.parametrize("rows", [640, 200])
def test_captured(rows):
    import ttperf
    torch = torch_mod()
    w, p = _table(500, 96, "mixed"), _table(64, 96, "mixed", 1)
    with B.store_of([w, p], "mixed") as store:
        store.set_stream(torch.cuda.Stream())
        torch.cuda.synchronize()
        t, at = _tokens(rows, 500, 1), _tokens(rows, 64, 2, "positions")
        dy = torch.randn(rows, 96, device="cuda").bfloat16()
        y = store.embedding(1, t, position=2, positions=at)
        store.accumulate_embedding_grad(1, t, dy)
        store.begin_capture()
        store.zero_grad(set_to_none=True)
        store.embedding(1, t, position=2, positions=at, out=y)
        store.accumulate_embedding_grad(1, t, dy)
        store.accumulate_embedding_grad(2, at, dy)
        store.accumulate_embedding_grad(1, t, dy, scale=0.5)
        graph = store.end_capture()
        for k in range(3):
            t.copy_(_tokens(rows, 500, 50 + k))
            torch.cuda.synchronize()
            graph.replay()
            store.sync()
            got = [v.clone() for v in (y, B.grad(store, 1), B.grad(store, 2))]
            store.zero_grad(set_to_none=True)
            e = store.embedding(1, t, position=2, positions=at)
            for i, ids, s in ((1, t, 1.0), (2, at, 1.0), (1, t, 0.5)):
                store.accumulate_embedding_grad(i, ids, dy, scale=s)
            store.sync()
            assert all(torch.equal(u.nan_to_num(), v.nan_to_num())
                       for u, v in zip(got, (e, B.grad(store, 1), B.grad(store, 2))))
        graph.close()
        store.begin_capture()
        with pytest.raises(ttperf.TTPError):
            store.accumulate_embedding_grad(1, t, dy)
        store.end_capture(discard=True)


def test_a_table_of_many_rows():
    """More rows than one launch has waves for their zeros."""
    import ttperf
    torch = torch_mod()
    vocab, cols = (1 << 24) + 1003, 4
    with ttperf.ParamStore([(vocab, cols)], mode="bf16") as store:
        store.torch_view(ttperf.BUF_GRAD).fill_(3.0)
        g = torch.Generator(device="cuda").manual_seed(4)
        t = torch.randperm(vocab, generator=g, device="cuda")[:700]
        t[:3] = torch.tensor([0, vocab - 1, (1 << 24) + 17], device="cuda")
        t = t.unique()
        dy = torch.randn(t.numel(), cols, generator=g, device="cuda").bfloat16()
        store.accumulate_embedding_grad(0, t, dy)
        grad = store.torch_view(ttperf.BUF_GRAD)[:vocab * cols].view(vocab, cols)
        assert torch.equal(grad[t], dy)
        grad[t] = 0
        assert not grad.any()


def test_a_table_past_2_to_the_32_elements():
    """Rows at the table's far end: lookup, gradient, zeros where no token is."""
    import ttperf
    torch = torch_mod()
    cols = 520
    vocab = 2 ** 32 // cols + 1000
    store = ttperf.ParamStore([(vocab, cols)], mode="bf16")
    store.set_stream(torch.cuda.current_stream())
    w = store.tensors[0].torch_view()
    t = torch.tensor([vocab - 1, 5, vocab - 1, 2 ** 32 // cols + 7, vocab], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.randn(5, cols, generator=g, device="cuda").bfloat16()
    w[t[:4]] = rows[:4]
    w[vocab - 1] = rows[2]
    y = store.embedding(0, t)
    assert torch.equal(y[1:4], rows[1:4]) and torch.equal(y[0], rows[2]) and y[4].isnan().all()
    grad = B.grad(store, 0)
    for more in (0, 600):  # tokens of padding: in one launch, and sorted
        grad[-2000:] = 9.0
        store.zero_grad(set_to_none=True, fill=False)
        store.accumulate_embedding_grad(0, torch.cat([t, t.new_full((more,), -1)]),
                                        torch.cat([rows, rows.new_ones(more, cols)]))
        assert torch.equal(grad[vocab - 1], (rows[0].float() + rows[2].float()).bfloat16())
        assert torch.equal(grad[t[1]], rows[1]) and torch.equal(grad[t[3]], rows[3])
        last = grad[-2000:].clone()
        last[t[3] - (vocab - 2000)] = 0
        assert (last[:-1] == 0).all()
    del w, grad
    store.close()


def test_refusals():
    import ttperf
    torch = torch_mod()
    with B.store_of([torch.zeros(30, 20, device="cuda"), torch.zeros(9, 21, device="cuda")],
                    "fp32") as store:
        t = _tokens(6, 30, 1, "uniform")
        dy = torch.zeros(6, 20, device="cuda")
        for bad in (dict(index=0), dict(index=7), dict(index=-1), dict(index=None),
                    dict(tokens=t.int()), dict(tokens=t.cpu()), dict(tokens=[1, 2]),
                    dict(scale=float("nan")), dict(scale=1e39), dict(position=2),
                    dict(positions=t), dict(position=2, positions=t),
                    dict(position=1, positions=t[:3]), dict(dtype=torch.float16),
                    dict(out=torch.empty(6, 21, device="cuda")),
                    dict(out=dy.bfloat16(), dtype=torch.float32)):
            a = dict(dict(index=1, tokens=t), **bad)
            with pytest.raises((ValueError, ttperf.TTPError)):
                store.embedding(a.pop("index"), a.pop("tokens"), **a)
        for bad in (dict(index=0), dict(index=7), dict(tokens=t[:5]), dict(tokens=t.int()),
                    dict(dy=dy[:, :19]), dict(dy=dy.half()), dict(scale=float("inf")),
                    dict(tokens=t.view(3, 2), dy=dy.view(2, 3, 20))):
            a = dict(dict(index=1, tokens=t, dy=dy), **bad)
            with pytest.raises((ValueError, ttperf.TTPError)):
                store.accumulate_embedding_grad(a.pop("index"), a.pop("tokens"), a.pop("dy"), **a)
        table = store.tensors[1].torch_view()
        with pytest.raises(ValueError, match="overlap"):
            store.embedding(1, t, out=table.view(30, 20)[:6])
        with pytest.raises(ValueError, match="overlap"):
            store.accumulate_embedding_grad(1, t, B.grad(store, 1)[:6])
        assert not any(store.has_grad(i) for i in range(4))
