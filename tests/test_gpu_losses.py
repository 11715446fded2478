"""GPU tests of the losses over logits (token_logprobs, preference_loss, policy_loss) against
plain forms in 64 bits, gradients by automatic differentiation of those and by differences.

Tolerances, from the arithmetic (u = 2^-24):
  logp   z_y - m and log s are rounded once each; s is a sum of V exponentials, at most V / 256 +
         20 additions deep, each exponential 2 units and its argument's rounding (|z - m| u log2 e)
         off, which the terms that matter (z near m) do not show:
         u (|z_y - m| + |log s| + V / 256 + 64)
  grad   c ([v = y] - p): p is off by the exponent's argument (|z_v - m| 3 u) and s; c by the
         rows' sums; rounded once to its type: 2^-8 relative in bf16, u in fp32
"""
import math

import pytest

from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _store(**kw):
    import ttperf
    torch = torch_mod()
    s = ttperf.ParamStore([(64,)], mode="mixed")
    s.set_stream(torch.cuda.current_stream())
    if kw.get("scale"):
        s.configure_scaler(True, init_scale=kw["scale"])
    return s


def _logits(rows, vocab, dtype, seed, pitch=0, offset=0):
    """Random logits as a view into a wider buffer (row pitch and first element's offset)."""
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch = max(pitch, vocab)
    buf = torch.full((rows * pitch + offset + 64,), 1e4, device="cuda").to(dtype)
    z = torch.as_strided(buf, (rows, vocab), (pitch, 1), offset)
    z.copy_((torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype))
    y = torch.randint(vocab, (rows,), generator=g, device="cuda")
    return z, y


def _logp64(z, y):
    """Log-probabilities in 64 bits on the host, by their definition (masked rows 0).  The row's
    maximum comes off first: at the type's lowest values z + log V is z again, also in 64 bits."""
    torch = torch_mod()
    z = z.detach().double().cpu() if not z.requires_grad else z
    y = y.cpu()
    top = z.detach().max(1, keepdim=True).values if len(z) else z.detach()
    z = z - torch.where(top.isfinite(), top, torch.zeros_like(top))
    lse = torch.logsumexp(z, 1)
    at = z.gather(1, y.clamp(min=0)[:, None])[:, 0]
    return torch.where(y >= 0, at - lse, torch.zeros((), dtype=torch.float64))


def _logp_tol(z, y):
    z = z.detach().double().cpu()
    m = z.max(1).values
    at = z.gather(1, y.cpu().clamp(min=0)[:, None])[:, 0]
    s = (z - m[:, None]).exp().sum(1)
    return U * ((at - m).abs() + s.log().abs() + z.shape[1] / 256 + 64)


def _check_grad(got, want, z, coef, dtype, c_err):
    """`coef`: the rows' |c| (or more); `c_err`: the rows' error of c.  c is a sum of terms that
    can cancel (an advantage's against the distance's), so its error is one of the terms'."""
    torch = torch_mod()
    got, z = got.double().cpu(), z.detach().double().cpu()
    far = (z.max(1, keepdim=True).values - z)
    rel = 2.0 ** -8 if dtype == torch.bfloat16 else 2 * U
    c, c_err = coef[:, None].clamp(min=1e-300), c_err[:, None]
    tol = want.abs() * (rel + c_err / c + U * (3 * far + z.shape[1] / 256 + 64))
    # at the token: the difference of c and c p, each with the errors above
    tol = tol + (c_err + c * U * (z.shape[1] / 256 + 64)) * \
        (want.abs() > 0) * ((want / c).abs() > 1e-3) + 1e-37
    bad = (got - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol).max()))


SHAPES = [(1, 1), (1, 2), (3, 7), (5, 8), (70, 65), (1, 50257), (2, 50257), (33, 4099),
          (300, 1000), (1100, 257), (9, 131077)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("pitch,offset", [(0, 0), (11, 3)])
def test_token_logprobs(rows, vocab, dtype, pitch, offset):
    torch = torch_mod()
    dt = getattr(torch, dtype)
    z, y = _logits(rows, vocab, dt, rows + vocab, pitch and vocab + pitch, offset)
    y[::3] = -100
    y[-1] = vocab - 1
    with _store() as store:
        got = store.token_logprobs(z, y)
        again = store.token_logprobs(z, y)
    assert got.shape == y.shape and got.dtype == torch.float32
    assert torch.equal(got, again)
    want = _logp64(z, y)
    assert ((got.double().cpu() - want).abs() <= _logp_tol(z, y)).all()
    assert (got[y < 0] == 0).all()


def test_token_logprobs_special_rows():
    """-inf logits (a masked vocabulary), rows that nothing is left of, infinities and NaN, a
    masked row that holds NaN, tokens past the vocabulary, the type's lowest value."""
    torch = torch_mod()
    for dt in (torch.bfloat16, torch.float32):
        for vocab in (5, 300, 50257):
            z = torch.randn(10, vocab, device="cuda").to(dt)
            low = torch.finfo(dt).min
            y = torch.full((10,), 2, device="cuda")
            z[0, 3:] = -math.inf          # part of the vocabulary ruled out
            z[1] = -math.inf              # all of it
            z[2, 2] = -math.inf           # the token itself
            z[3, 1] = math.inf
            z[4, 4] = math.nan
            z[5] = math.nan
            y[5] = -1                     # masked: not read
            y[6] = vocab                  # past the end
            y[7] = 2 ** 40
            z[8, :2] = low
            z[8, 3:] = low                # the type's lowest value where a mask puts it
            z[9] = low
            with _store() as store:
                got = store.token_logprobs(z, y).double().cpu()
            want = _logp64(z, torch.where(y >= vocab, 0, y))
            assert got[5] == 0 and got[2] == -math.inf and got[8] == 0
            for r in (1, 3, 4, 6, 7):
                assert math.isnan(got[r]), (r, got[r])
            for r in (0, 9):
                assert abs(got[r] - want[r]) <= U * (abs(want[r]) + vocab / 256 + 64), r


def _preference64(z, y, starts, ref, beta, eps):
    torch = torch_mod()
    logp = _logp64(z, y)
    live = (y >= 0).cpu()
    d = torch.where(live, logp - (0 if ref is None else ref.double().cpu()),
                    torch.zeros((), dtype=torch.float64))
    at, pairs = starts.tolist(), starts.numel() // 2
    at = [min(max(a, 0), z.shape[0]) for a in at]
    total = torch.stack([d[a:b].sum() for a, b in zip(at, at[1:])])
    h = beta * (total[:pairs] - total[pairs:])
    sig = torch.sigmoid
    loss = (-(1 - eps) * torch.log(sig(h)) - eps * torch.log(sig(-h))).mean()
    return loss, h, logp, d


@pytest.mark.parametrize("rows,vocab,pairs", [(0, 7, 1), (2, 3, 1), (41, 65, 3), (200, 1001, 17),
                                              (37, 50257, 2), (1300, 130, 40)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("eps,with_ref,scale", [(0.0, True, 0.0), (0.1, False, 512.0)])
def test_preference_loss(rows, vocab, pairs, dtype, eps, with_ref, scale):
    torch = torch_mod()
    dt = getattr(torch, dtype)
    z, y = _logits(rows, vocab, dt, 7 * rows + vocab, vocab + 3, 1)
    y[::4] = -100
    g = torch.Generator().manual_seed(rows)
    cuts = torch.randint(0, rows + 1, (2 * pairs + 1,), generator=g).sort().values
    if rows > 40:  # some rows before the first and behind the last sequence, an empty sequence
        cuts[0], cuts[-1], cuts[1] = 2, rows - 3, 2
        cuts = cuts.sort().values
    starts = cuts.cuda()
    # a reference near the model: margins of order one
    ref = None
    if with_ref:
        ref = (_logp64(z, y) + 0.3 * torch.randn(rows, generator=g)).float().cuda()
    with _store(scale=scale) as store:
        r = store.preference_loss(z, y, starts, ref, beta=0.13, label_smoothing=eps)
        only = store.preference_loss(z, y, starts, ref, beta=0.13, label_smoothing=eps,
                                     grad=False)
        assert only.grad is None
        for a, b in zip(r[:3], only[:3]):
            assert torch.equal(a, b)
        twin = z.clone()  # in the logits' place
        same = store.preference_loss(twin, y, starts, ref, beta=0.13, label_smoothing=eps,
                                     grad=twin)
        assert same.grad is twin and torch.equal(twin, r.grad)
    z64 = z.double().cpu().requires_grad_()
    loss, h, logp, d = _preference64(z64, y, starts, ref, 0.13, eps)
    (loss * (scale or 1)).backward()
    tol = _logp_tol(z, y)
    assert ((r.logps.double().cpu() - logp).abs() <= tol).all()
    # a margin: the rows' errors, at worst all of one sign, and its own rounding
    h_tol = 0.13 * float(tol.sum()) + 2 * U * h.abs().max() + 1e-12
    assert ((r.margins.double().cpu() - h).abs() <= h_tol).all()
    assert abs(float(r.loss) - loss.item()) <= float(h_tol) + 2 * U * abs(loss.item())
    want = torch.zeros_like(z64) if z64.grad is None else z64.grad
    coef = want.abs().max(1).values * 2 if rows else want.sum(1)
    if rows:
        _check_grad(r.grad, want, z, coef, dt, coef * (float(h_tol) + 4 * U))
    # masked rows and rows of no sequence: exact zeros
    outside = torch.ones(rows, dtype=torch.bool)
    outside[int(starts[0]):int(starts[-1])] = False
    assert (r.grad.cpu()[outside | (y < 0).cpu()] == 0).all()


@pytest.mark.parametrize("rows,vocab,pairs", [(4096, 65, 2), (4096, 65, 16), (4096, 65, 17),
                                              (4097, 65, 16), (300, 9000, 16), (300, 9000, 17)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_preference_loss_where_its_launches_change(rows, vocab, pairs, dtype):
    """Few pairs over few rows are finished by the last block of the launch that scores the rows,
    or of the one that joins their parts; more by a launch of their own."""
    test_preference_loss(rows, vocab, pairs, dtype, 0.1, True, 512.0)


def _policy64(z, y, old, adv, ref, low, high, k_coef, denom):
    torch = torch_mod()
    logp = _logp64(z, y)
    live = (y >= 0).cpu()
    r = torch.exp(logp - old.double().cpu())
    a = adv.double().cpu()
    loss = -torch.minimum(r * a, r.clamp(1 - low, 1 + high) * a)
    kl = torch.zeros_like(loss)
    if ref is not None:
        gap = ref.double().cpu() - logp
        kl = torch.exp(gap) - gap - 1
    n = denom or max(int(live.sum()), 1)
    zero = torch.zeros((), dtype=torch.float64)
    return (torch.where(live, loss + k_coef * kl, zero).sum() / n,
            torch.where(live, kl, zero).sum() / n, logp)


@pytest.mark.parametrize("rows,vocab", [(0, 5), (1, 1), (1, 50257), (3, 70), (129, 65),
                                        (260, 4100), (40, 50257), (700, 333), (5, 131077),
                                        (2, 270001)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("kl,scale,denom", [(0.0, 0.0, None), (0.05, 1024.0, None),
                                            (0.05, 0.0, 77.0)])
def test_policy_loss(rows, vocab, dtype, kl, scale, denom):
    torch = torch_mod()
    dt = getattr(torch, dtype)
    z, y = _logits(rows, vocab, dt, 3 * rows + vocab, vocab + (5 if vocab % 2 else 0), 2)
    y[1::4] = -1
    g = torch.Generator().manual_seed(rows + vocab)
    base = _logp64(z, y)
    old = (base + 0.3 * torch.randn(rows, generator=g)).float().cuda()
    adv = torch.randn(rows, generator=g).cuda()
    ref = (base + 0.3 * torch.randn(rows, generator=g)).float().cuda() if kl else None
    args = (y, old, adv, ref)
    kw = dict(clip=(0.2, 0.3), kl_coef=kl, denominator=denom)
    with _store(scale=scale) as store:
        r = store.policy_loss(z, *args, **kw)
        only = store.policy_loss(z, *args, grad=False, **kw)
        for a, b in zip(r[:3], only[:3]):
            assert torch.equal(a, b)
        twin = z.clone()
        same = store.policy_loss(twin, *args, grad=twin, **kw)
        assert torch.equal(twin, r.grad) and torch.equal(same.loss, r.loss)
    z64 = z.double().cpu().requires_grad_()
    loss, mean_kl, logp = _policy64(z64, *args, 0.2, 0.3, kl, denom)
    (loss * (scale or 1)).backward()
    if not rows:
        assert float(r.loss) == 0 and float(r.kl) == 0
        return
    tol = _logp_tol(z, y)
    assert ((r.logps.double().cpu() - logp).abs() <= tol).all()
    # r and exp(g) move by the error of logp, relative, and a few units of the exponentials
    e = float(tol.max()) + 8 * U
    assert abs(float(r.loss) - loss.item()) <= 4 * e * (abs(loss.item()) + 4)
    assert abs(float(r.kl) - mean_kl.item()) <= 4 * e * (abs(mean_kl.item()) + 1)
    n = (denom or max(int((y >= 0).sum()), 1)) / (scale or 1)
    a = (adv.double().cpu() * torch.exp(logp - old.double().cpu())).abs() / n
    b = kl * torch.exp(ref.double().cpu() - logp) / n if kl else 0 * a
    c = z64.grad.abs().max(1).values
    # the largest element of a row is c (1 - p_y), or c p_v of another one: |c| is its sum / 2
    c = torch.maximum(c, z64.grad.abs().sum(1) / 2)
    _check_grad(r.grad, z64.grad, z, c, dt, 4 * e * (a + b))
    assert (r.grad[y < 0] == 0).all()


@pytest.mark.parametrize("rows", [2047, 2048, 2049])
@pytest.mark.parametrize("vocab", [65, 2500])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_policy_loss_where_its_launches_change(rows, vocab, dtype):
    """Few rows are counted and summed by the launch that makes the gradient, more by their own:
    the same numbers from either (the last rows masked: their logits are not the difference)."""
    torch = torch_mod()
    z, y = _logits(rows, vocab, getattr(torch, dtype), rows, 0, 0)
    y[::5] = -1
    y[2040:] = -1
    g = torch.Generator().manual_seed(rows)
    base = _logp64(z, y)
    old = (base + 0.3 * torch.randn(rows, generator=g)).float().cuda()
    adv = torch.randn(rows, generator=g).cuda()
    with _store(scale=256.0) as store:
        r = store.policy_loss(z, y, old, adv, old, kl_coef=0.1)
        more = [torch.cat([t, t[-1:].expand(3, *t.shape[1:])]) for t in (z, y, old, adv)]
        m = store.policy_loss(*more, more[2], kl_coef=0.1)
    loss, mean_kl, logp = _policy64(z, y, old, adv, old, 0.2, 0.2, 0.1, None)
    e = float(_logp_tol(z, y).max()) + 8 * U
    assert abs(float(r.loss) - loss.item()) <= 4 * e * (abs(loss.item()) + 4)
    assert abs(float(r.kl) - mean_kl.item()) <= 4 * e * (abs(mean_kl.item()) + 1)
    assert torch.equal(m.grad[:rows], r.grad) and torch.equal(m.logps[:rows], r.logps)
    # the sums are in 64 bits, in another order
    assert abs(float(m.loss) - float(r.loss)) <= 2 * U * abs(float(r.loss))
    assert abs(float(m.kl) - float(r.kl)) <= 2 * U * abs(float(r.kl))


def test_policy_loss_without_a_row_that_counts():
    """All rows masked, their logits NaN: loss 0, gradient 0."""
    torch = torch_mod()
    for vocab in (65, 50257):
        z = torch.full((4, vocab), math.nan, device="cuda", dtype=torch.bfloat16)
        y = torch.full((4,), -100, device="cuda")
        v = torch.full((4,), math.nan, device="cuda")
        with _store() as store:
            r = store.policy_loss(z, y, v, v, v, kl_coef=0.1)
            p = store.preference_loss(z, y, torch.tensor([0, 2, 4], device="cuda"), v)
        assert float(r.loss) == 0 and float(r.kl) == 0 and (r.grad == 0).all()
        assert abs(float(p.loss) - math.log(2)) < 1e-6 and (p.grad == 0).all()
        assert (r.logps == 0).all() and (p.logps == 0).all()


def test_what_is_not_finite_reaches_the_loss_and_the_gradient():
    """A NaN or a token past the vocabulary on a row that counts is not lost: the loss is NaN, and
    so are the gradients that depend on it (a step with loss scaling then skips)."""
    torch = torch_mod()
    for dt in (torch.float32, torch.bfloat16):
        for vocab in (65, 50257):
            z = torch.randn(6, vocab, device="cuda").to(dt)
            y = torch.tensor([1, 2, 3, 4, 5, vocab + 3], device="cuda")
            z[1, 5] = math.nan
            zero = torch.zeros(6, device="cuda")
            with _store() as store:
                r = store.policy_loss(z, y, zero - 3, zero + 1, zero - 3, kl_coef=0.1)
                p = store.preference_loss(z, y, torch.tensor([0, 2, 3, 4, 6], device="cuda"))
            assert math.isnan(float(r.loss)) and math.isnan(float(p.loss))
            assert r.grad[1].isnan().all() and r.grad[5].isnan().all()
            assert r.grad[[0, 2, 3, 4]].isfinite().all()
            assert p.grad[[0, 1, 3, 4, 5]].float().isnan().any(1)[:2].all()
            # a clipped or zero-advantage row with a part of its vocabulary ruled out stays finite
            z = torch.randn(2, vocab, device="cuda").to(dt)
            z[:, 7:] = -math.inf
            y = torch.tensor([1, 2], device="cuda")
            with _store() as store:
                r = store.policy_loss(z, y, zero[:2] - 2, zero[:2] + 1)
            assert r.grad.isfinite().all() and (r.grad[:, 7:] == 0).all()


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_gradient_against_differences(kind):
    """Central differences of the loss in fp32 logits: the loss's own error (4e-6) over twice the
    step (0.02) bounds the difference quotient's, with the third derivative's h^2 part."""
    torch = torch_mod()
    z, y = _logits(6, 9, torch.float32, 5)
    z = z.contiguous()
    y[2] = -100
    old = _logp64(z, y).float().cuda() + 0.05
    adv = torch.tensor([1.0, -1, 2, 0.5, -0.5, 1], device="cuda")
    starts = torch.tensor([0, 2, 3, 5, 6], device="cuda")
    h = 0.02
    with _store() as store:
        def loss(x, grad):
            if kind == "policy":
                return store.policy_loss(x, y, old, adv, old, clip=(0.5, 0.5), kl_coef=0.3,
                                         grad=grad)
            return store.preference_loss(x, y, starts, old, beta=0.7, label_smoothing=0.1,
                                         grad=grad)
        g = loss(z, True).grad
        for r in range(6):
            for v in range(9):
                up, down = z.clone(), z.clone()
                up[r, v] += h
                down[r, v] -= h
                num = (float(loss(up, False).loss) - float(loss(down, False).loss)) / (2 * h)
                assert abs(num - float(g[r, v])) <= 4e-6 / (2 * h) + 2 * h * h, (r, v)


def test_a_batch_of_sequences_keeps_its_shape():
    """(B, T, V) logits and (B, T) targets; the gradient goes on through torch's backward."""
    torch = torch_mod()
    z = torch.randn(4, 6, 33, device="cuda", requires_grad=True)
    y = torch.randint(33, (4, 6), device="cuda")
    with _store() as store:
        r = store.preference_loss(z, y, torch.arange(0, 25, 6, device="cuda"))
        assert r.logps.shape == (4, 6) and r.grad.shape == z.shape
        z.backward(r.grad)
        assert torch.equal(z.grad, r.grad)
        assert store.token_logprobs(z, y).equal(r.logps)


def test_on_the_stores_own_stream():
    """Inputs made on torch's stream, the store on another: each waits for the other."""
    torch = torch_mod()
    import ttperf
    store = ttperf.ParamStore([(64,)], mode="mixed")  # its own stream
    shared = _store()
    for k in range(3):
        z = torch.randn(512, 5003, device="cuda", dtype=torch.bfloat16)
        for _ in range(8):
            z = z * 1.01
        y = torch.randint(5003, (512,), device="cuda")
        got = store.token_logprobs(z, y) * 1.0
        assert torch.equal(got, shared.token_logprobs(z, y))
    store.close()
    shared.close()


def test_captured_losses():
    """Captured once, replayed several times with other logits and a moved loss scale, eager work
    between the replays."""
    torch = torch_mod()
    import ttperf
    s = torch.cuda.Stream()
    store = ttperf.ParamStore([(64,)], mode="mixed")
    store.set_stream(s)
    store.configure_scaler(True, init_scale=64.0)
    eager = _store(scale=64.0)
    for rows, vocab in ((9, 50257), (700, 600)):
        with torch.cuda.stream(s):
            z, y = _logits(rows, vocab, torch.bfloat16, 3)
            z = z.contiguous()
            y[::5] = -1
            v = -torch.rand(rows, device="cuda") * 9
            starts = torch.tensor([0, 2, 5, 6, rows], device="cuda")
            r = store.policy_loss(z, y, v, v, v, kl_coef=0.1)
            p = store.preference_loss(z, y, starts, v)
            t = store.token_logprobs(z, y)
            store.sync()
            store.begin_capture()
            with pytest.raises(ValueError):
                store.token_logprobs(z, y)
            store.policy_loss(z, y, v, v, v, kl_coef=0.1, out=r)
            store.preference_loss(z, y, starts, v, out=p)
            store.token_logprobs(z, y, out=t)
            graph = store.end_capture()
        for k in range(4):
            with torch.cuda.stream(s):
                z.copy_(torch.randn(rows, vocab, device="cuda"))
                store.set_scaler_state(64.0 * (k + 1), 0)
                graph.replay()
                torch.cuda.synchronize()
            eager.set_scaler_state(64.0 * (k + 1), 0)
            a = eager.policy_loss(z, y, v, v, v, kl_coef=0.1)
            b = eager.preference_loss(z, y, starts, v)
            for x, w in list(zip(r, a)) + list(zip(p, b)) + [(t, a.logps)]:
                assert torch.equal(x, w)
        graph.close()
    store.close()
    eager.close()


def test_refusals():
    import ttperf
    torch = torch_mod()
    z = torch.randn(8, 20, device="cuda")
    y = torch.randint(20, (8,), device="cuda")
    v = torch.zeros(8, device="cuda")
    starts = torch.tensor([0, 4, 8], device="cuda")
    with _store() as store:
        def refused(call, exc=ValueError):
            with pytest.raises(exc):
                call()
        refused(lambda: store.token_logprobs(z.cpu(), y))
        refused(lambda: store.token_logprobs(z.double(), y))
        refused(lambda: store.token_logprobs(z, y.int()))
        refused(lambda: store.token_logprobs(z, y[:7]))
        refused(lambda: store.token_logprobs(z.t(), y[:1].expand(20)))
        refused(lambda: store.token_logprobs(z[:1].expand(8, 20), y))
        refused(lambda: store.token_logprobs(z[:, :0], y))
        refused(lambda: store.token_logprobs(z, y, out=v.double()))
        refused(lambda: store.token_logprobs(z, y, out=z.view(-1)[:8]))  # overlaps the logits
        refused(lambda: store.preference_loss(z, y, starts[:2]))
        refused(lambda: store.preference_loss(z, y, starts, beta=0.0))
        refused(lambda: store.preference_loss(z, y, starts, beta=float("nan")))
        refused(lambda: store.preference_loss(z, y, starts, label_smoothing=0.6))
        refused(lambda: store.preference_loss(z, y, starts, v[:3]))
        refused(lambda: store.preference_loss(z, y, starts, grad=z.bfloat16()))
        refused(lambda: store.preference_loss(z, y, starts, grad=torch.empty(8, 21, device="cuda")))
        wide = torch.randn(9, 20, device="cuda")
        refused(lambda: store.preference_loss(wide[:8], y, starts, grad=wide[1:]))  # shifted
        refused(lambda: store.policy_loss(z, y, v, v, clip=(-0.1, 0.2)))
        refused(lambda: store.policy_loss(z, y, v, v, clip=(0.2, -0.1)))
        refused(lambda: store.policy_loss(z, y, v, v, kl_coef=-1.0))
        refused(lambda: store.policy_loss(z, y, v, v, kl_coef=0.1))  # no reference
        refused(lambda: store.policy_loss(z, y, v, v, denominator=0.0))
        refused(lambda: store.policy_loss(z, y, v, v.double()))
        # columns of one wider buffer side by side do not overlap
        both = torch.randn(8, 40, device="cuda")
        left, right = both[:, :20], both[:, 20:]
        r = store.preference_loss(left, y, starts, grad=right)
        assert torch.equal(right, store.preference_loss(left.contiguous(), y, starts).grad)
        assert r.grad is right
        assert isinstance(ttperf.TTPValueError(-1, ""), ValueError)
