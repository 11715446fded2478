"""GPU tests of activations kept in 8 bits: the format bit by bit against its definition, GELU and
its gradient from the kept values against 64 bits.

Tolerances: the kept values and scales are exact (a power-of-two scale, one rounding).  GELU's
distribution function is 2e-7 off at most (its polynomial 2.3e-8, half of 4.5e-8 of erfc, the rest
fp32 arithmetic; relative to itself: tests/test_gpu_gelu_tail.py): 4e-7 |x| for x Phi(x); the tanh form's quotient has the exponential
and the reciprocal (1 unit each) and its argument 2 u with |2 u| 4 2^-24 of error that counts
while s (1 - s) |2 u| < 0.6: 1e-6 |x|.  The slope has the same errors with |x| dphi <= 1.2 in the
place of x: 1e-6 |dy| (1 + |x|).  Each is rounded once to its type: 2^-8 relative in bf16 (8
significant bits), 2^-24 in fp32."""
import math

import numpy as np
import pytest

from gpu_util import torch_mod

pytestmark = pytest.mark.gpu


def _store(**kw):
    import ttperf
    torch = torch_mod()
    s = ttperf.ParamStore([(64,)], mode="mixed")
    s.set_stream(torch.cuda.current_stream())
    return s


def _view(x, pitch, offset):
    """x as a view with the given row pitch and first element's offset."""
    torch = torch_mod()
    rows, cols = x.shape
    pitch = max(pitch, cols)
    buf = torch.full((rows * pitch + offset + 16,), 7e4, device="cuda", dtype=x.dtype)
    v = torch.as_strided(buf, (rows, cols), (pitch, 1), offset)
    v.copy_(x)
    return v, buf


def _e4m3_grid():
    """The magnitudes of fp8 e4m3 in order, by its definition (index = the code)."""
    out = []
    for code in range(127):  # 0x7F is NaN
        e, m = code >> 3, code & 7
        out.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return np.array(out)


def _kept64(x, fmt):
    """(values as numbers, scale bytes) by the definition, on the host in 64 bits."""
    rows, cols = x.shape
    width = -(-cols // 32) * 32
    b = np.zeros((rows, width))
    b[:, :cols] = x.double().cpu().numpy()
    b = b.reshape(rows, -1, 32)
    most, least = (127, 1) if fmt == "int8" else (448, 10)
    top = np.abs(b).max(2)
    finite = np.isfinite(b).all(2)
    scale = np.full(top.shape, 255)
    for r, k in np.ndindex(*top.shape):
        if finite[r, k]:
            e = least
            while math.ldexp(most, e - 127) < top[r, k]:
                e += 1
            scale[r, k] = e
    with np.errstate(invalid="ignore", over="ignore"):
        v = np.ldexp(b, (127 - scale)[:, :, None])
    v[~finite] = 0
    if fmt == "int8":
        v = np.rint(v)
    else:
        grid = _e4m3_grid()
        a = np.abs(v)
        hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
        lo = hi - 1
        up = (a - grid[lo] > grid[hi] - a) | ((a - grid[lo] == grid[hi] - a) & (hi % 2 == 0))
        v = np.copysign(np.where(up, grid[hi], grid[lo]), v)
    return v.reshape(rows, width), scale


def _as_numbers(kept):
    torch = torch_mod()
    v = kept.values.cpu()
    v = v.view(torch.int8).double() if kept.format == "int8" else \
        v.view(torch.float8_e4m3fn).double()
    return v.numpy()


SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (2, 8), (7, 65), (130, 100), (257, 384), (64, 1537)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("pitch,offset", [(0, 0), (5, 3)])
def test_pack_and_restore(rows, cols, dtype, fmt, pitch, offset):
    torch = torch_mod()
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(rows * cols)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    # magnitudes over the whole range of exponents, block by block, and zero blocks
    x *= torch.exp2(torch.randint(-30, 30, (rows, -(-cols // 32)), generator=g,
                                  device="cuda").float()).repeat_interleave(32, 1)[:, :cols]
    x[:, ::5] = 0
    x[-1, :32] = 0
    x, _ = _view(x.to(dt), pitch and cols + pitch, offset)
    with _store() as store:
        kept = store.checkpoint8(x, fmt=fmt)
        back = store.restore8(kept)
        wide = store.restore8(kept, dtype=torch.float32)
        out, buf = _view(torch.zeros_like(x), cols + 3, 1)
        before = buf.clone()
        narrow = store.restore8(kept, out=torch.empty(rows, cols, device="cuda",
                                                      dtype=torch.bfloat16))
    v, scale = _kept64(x, fmt)
    assert (kept.scales.cpu().numpy() == scale).all()
    got = _as_numbers(kept)
    assert (got == v).all()
    want = np.ldexp(v, np.repeat(scale, 32, 1) - 127)[:, :cols]
    for b in (back, wide, narrow):
        assert (b.double().cpu().numpy() == want).all()
    assert back.dtype == dt and torch.equal(buf, before)
    assert abs(want - x.double().cpu().numpy()).max() <= \
        np.abs(x.double().cpu().numpy()).max() * (2.0 ** -7 if fmt == "int8" else 2.0 ** -4)


def test_every_rounding_tie_and_boundary():
    """Values on, between and next to the grid's points, and scales at a mantissa's boundary."""
    torch = torch_mod()
    for fmt, most in (("int8", 127.0), ("e4m3", 448.0)):
        grid = np.arange(0, 128) if fmt == "int8" else _e4m3_grid()
        mid = (grid[1:] + grid[:-1]) / 2
        pts = np.concatenate([grid, mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                              np.nextafter(mid.astype(np.float32), np.float32(1e9))])
        pts = np.concatenate([pts, -pts]).astype(np.float32)
        pts = pts[np.abs(pts) <= most]
        pts = np.resize(pts, (-(-len(pts) // 31), 31))
        x = np.concatenate([np.full((len(pts), 1), most, np.float32), pts], 1)
        above = np.zeros((4, 32), np.float32)
        above[:, 0] = [most, np.nextafter(np.float32(most), np.float32(1e9)), most * 2, most / 2]
        above[:, 1:] = np.random.default_rng(3).normal(0, most / 3, (4, 31)).astype(np.float32)
        x = torch.from_numpy(np.concatenate([x, np.clip(above, -most, None)]))
        for power in (-60, 0, 100):
            y = (x * 2.0 ** power).cuda()
            with _store() as store:
                kept = store.checkpoint8(y, fmt=fmt)
            v, scale = _kept64(y, fmt)
            assert (kept.scales.cpu().numpy() == scale).all()
            assert (_as_numbers(kept) == v).all()


def test_extremes_of_the_range():
    """The largest and least numbers, subnormals, infinities and NaN: a block that is not finite
    stands for NaN, the blocks beside it do not."""
    torch = torch_mod()
    for dt in (torch.float32, torch.bfloat16):
        for fmt in ("int8", "e4m3"):
            x = torch.zeros(8, 96, device="cuda")
            x[0] = torch.finfo(dt).max
            x[1] = -torch.finfo(dt).max
            x[2] = torch.finfo(dt).tiny
            x[3] = torch.finfo(dt).tiny / 64
            x[4, 40] = math.inf
            x[5, 95] = -math.inf
            x[6, 32] = math.nan
            x[7] = 1e-37
            x[4:7, 3] = 5.0
            x = x.to(dt)
            with _store() as store:
                kept = store.checkpoint8(x, fmt=fmt)
                back = store.restore8(kept, dtype=torch.float32).cpu()
            v, scale = _kept64(x, fmt)
            assert (kept.scales.cpu().numpy() == scale).all()
            assert (_as_numbers(kept) == v).all()
            bad = torch.zeros(8, 96, dtype=torch.bool)
            bad[4, 32:64] = bad[5, 64:] = bad[6, 32:64] = True
            assert torch.equal(back.isnan(), bad)


def _gelu64(x, approximate):
    torch = torch_mod()
    x = x.double().cpu().requires_grad_()
    if approximate == "tanh":
        y = x / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    else:
        y = x * torch.special.ndtr(x)
    (slope,) = torch.autograd.grad(y.sum(), x)
    return y.detach(), slope


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (17, 100), (257, 384), (40, 1537)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("approximate", ["none", "tanh"])
def test_gelu(rows, cols, dtype, fmt, approximate):
    torch = torch_mod()
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda") * 3
    x[:, ::7] = torch.linspace(-14, 14, len(x[0, ::7]), device="cuda")
    x, _ = _view(x.to(dt), cols + 3, 1)
    dy = torch.randn(rows, cols, generator=g, device="cuda").to(dt)
    with _store() as store:
        y, kept = store.gelu_checkpoint8(x, fmt=fmt, approximate=approximate)
        plain = store.checkpoint8(x, fmt=fmt)
        assert torch.equal(kept.values, plain.values) and torch.equal(kept.scales, plain.scales)
        dx = store.gelu_backward8(kept, dy, approximate=approximate)
        kx = store.restore8(kept, dtype=torch.float32)
        # in the input's and the gradient's places
        twin, gy = x.clone(), dy.clone()
        y2, _ = store.gelu_checkpoint8(twin, fmt=fmt, approximate=approximate, out=twin)
        assert y2 is twin and torch.equal(twin, y)
        store.gelu_backward8(kept, gy, approximate=approximate, out=gy)
        assert torch.equal(gy, dx)
    rel = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -24
    want, _ = _gelu64(x, approximate)
    tol = 1e-6 * x.double().cpu().abs() + rel * want.abs() + 1e-37
    assert ((y.double().cpu() - want).abs() <= tol).all()
    _, slope = _gelu64(kx, approximate)
    d64 = dy.double().cpu()
    want = d64 * slope
    tol = 1e-6 * d64.abs() * (1 + kx.double().cpu().abs()) + rel * want.abs() + 1e-37
    assert ((dx.double().cpu() - want).abs() <= tol).all()


def test_gelu_special_values():
    """Where a form saturates, overflows or is not finite: as the 64-bit form."""
    torch = torch_mod()
    x = torch.zeros(10, 32, device="cuda")
    x[:9, 0] = torch.tensor([math.inf, -math.inf, math.nan, 1e30, -1e30, 3e38, -3e38, 60., -60.])
    for approximate in ("none", "tanh"):
        with _store() as store:
            y, kept = store.gelu_checkpoint8(x, approximate=approximate)
            dx = store.gelu_backward8(kept, torch.ones_like(x), approximate=approximate)
        assert y[0, 0] == math.inf and y[1:3, 0].isnan().all()
        assert torch.equal(y[3:9, 0].abs(), torch.where(x[3:9, 0] > 0, x[3:9, 0], 0.0))
        assert (y[:, 1:] == 0).all()
        assert dx[:3].isnan().all()  # a block that is not finite stands for NaN
        assert torch.equal(dx[3:9, 0], (x[3:9, 0] > 0).float())
        assert (dx[3:, 1:] == 0.5).all() and (dx[9] == 0.5).all()


def test_gelu_gradient_against_differences():
    """Central differences of the forward at the kept values: its error 1e-6 (1 + |x|) over twice
    the step, and the third derivative's (below 2) h^2 / 6."""
    torch = torch_mod()
    h = 0.02
    for approximate in ("none", "tanh"):
        x = torch.linspace(-6, 6, 512, device="cuda").view(4, 128)
        with _store() as store:
            _, kept = store.gelu_checkpoint8(x, approximate=approximate)
            kx = store.restore8(kept)
            up, _ = store.gelu_checkpoint8(kx + h, approximate=approximate)
            down, _ = store.gelu_checkpoint8(kx - h, approximate=approximate)
            dx = store.gelu_backward8(kept, torch.ones_like(x), approximate=approximate)
        num = (up - down) / (2 * h)
        assert ((num - dx).abs() <= 2e-6 * (1 + kx.abs()) / (2 * h) + 2 * h * h / 6).all()


def test_empty_and_batched_shapes():
    torch = torch_mod()
    with _store() as store:
        x = torch.empty(0, 40, device="cuda")
        kept = store.checkpoint8(x)
        assert store.restore8(kept).shape == (0, 40)
        y, kept = store.gelu_checkpoint8(x)
        assert store.gelu_backward8(kept, x).shape == (0, 40) and y.shape == (0, 40)
        x = torch.randn(2, 3, 40, device="cuda", dtype=torch.bfloat16)
        y, kept = store.gelu_checkpoint8(x, approximate="tanh")
        assert y.shape == x.shape and kept.shape == (2, 3, 40)
        assert store.restore8(kept).shape == x.shape
        one = store.checkpoint8(x[0, 0])
        assert torch.equal(store.restore8(one), store.restore8(kept)[0, 0])


def test_captured():
    torch = torch_mod()
    import ttperf
    s = torch.cuda.Stream()
    store = ttperf.ParamStore([(64,)], mode="mixed")
    store.set_stream(s)
    eager = _store()
    with torch.cuda.stream(s):
        x = torch.randn(50, 130, device="cuda")
        y, kept = store.gelu_checkpoint8(x)
        dx = store.gelu_backward8(kept, x)
        store.sync()
        store.begin_capture()
        with pytest.raises(ValueError):
            store.checkpoint8(x)
        store.gelu_checkpoint8(x, out=y, kept=kept)
        store.gelu_backward8(kept, x, out=dx)
        graph = store.end_capture()
        for k in range(4):
            x.copy_(torch.randn(50, 130, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            want, wk = eager.gelu_checkpoint8(x)
            torch.cuda.synchronize()
            assert torch.equal(want, y) and torch.equal(wk.values, kept.values)
            assert torch.equal(wk.scales, kept.scales)
    graph.close()
    store.close()
    eager.close()


def test_refusals():
    torch = torch_mod()
    import ttperf
    x = torch.randn(6, 64, device="cuda")
    with _store() as store:
        kept = store.checkpoint8(x)

        def refused(call):
            with pytest.raises(ValueError):
                call()
        refused(lambda: store.checkpoint8(x, fmt="int4"))
        refused(lambda: store.checkpoint8(x.half()))
        refused(lambda: store.checkpoint8(x.t()))
        refused(lambda: store.checkpoint8(x.cpu()))
        refused(lambda: store.checkpoint8(x, out=store.checkpoint8(x[:5])))
        refused(lambda: store.checkpoint8(x, fmt="e4m3", out=kept))
        refused(lambda: store.restore8(x))
        refused(lambda: store.restore8(kept, dtype=torch.float16))
        refused(lambda: store.restore8(kept, out=torch.empty(6, 65, device="cuda")))
        refused(lambda: store.gelu_checkpoint8(x, approximate="fast"))
        refused(lambda: store.gelu_checkpoint8(x, out=x.bfloat16()))
        refused(lambda: store.gelu_backward8(kept, x[:5]))
        refused(lambda: store.gelu_backward8(kept, x, out=torch.empty(6, 63, device="cuda")))
        wide = torch.randn(7, 64, device="cuda")
        refused(lambda: store.gelu_checkpoint8(wide[:6], out=wide[1:]))  # shifted by a row
        # another activation's type: what is restored would have it
        refused(lambda: store.checkpoint8(x.bfloat16(), out=kept))
        refused(lambda: store.gelu_checkpoint8(x.bfloat16(), kept=kept))
        # kept memory of other sizes or types
        refused(lambda: ttperf.Checkpoint8(kept.values[:5], kept.scales, (6, 64), x.dtype, "int8"))
        refused(lambda: ttperf.Checkpoint8(kept.values, kept.scales[:, :1], (6, 64), x.dtype,
                                           "int8"))
        refused(lambda: ttperf.Checkpoint8(kept.values.int(), kept.scales, (6, 64), x.dtype,
                                           "int8"))
        # kept memory that overlaps, or is not aligned
        flat = torch.zeros(6 * 64 + 64, dtype=torch.uint8, device="cuda")
        off = ttperf.Checkpoint8(flat[8:8 + 384].view(6, 64), kept.scales, (6, 64), x.dtype,
                                 "int8")
        refused(lambda: store.checkpoint8(x, out=off))
        same = ttperf.Checkpoint8(flat[:384].view(6, 64), flat[372:384].view(6, 2), (6, 64),
                                  x.dtype, "int8")
        refused(lambda: store.checkpoint8(x, out=same))
