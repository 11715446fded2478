"""GPU tests of the policy loss at the longest row of each of its one-pass shapes, on and off the
16-byte grid, with tokens in a row's first, last and remaining columns.

Tolerances as in tests/test_gpu_losses.py."""
import pytest

from gpu_util import torch_mod
from test_gpu_losses import U, _check_grad, _logits, _logp_tol, _policy64, _store

pytestmark = pytest.mark.gpu

# 16-byte chunks of the longest row: lanes x chunks per lane (256 x 28 off the grid alone); one
# more chunk takes the next shape, behind the last one two passes
LIMITS = [64, 64 * 4, 256 * 4, 256 * 8, 256 * 16, 256 * 28, 1024 * 8, 1024 * 12, 1024 * 16,
          1024 * 20]


@pytest.mark.parametrize("limit", LIMITS)
@pytest.mark.parametrize("more", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("on_grid", [True, False])
def test_the_longest_row_of_a_shape(limit, more, dtype, on_grid):
    torch = torch_mod()
    dt = getattr(torch, dtype)
    per = 8 if dtype == "bfloat16" else 4
    chunks = limit + more
    vocab = chunks * per + per - 1  # a remainder of all but one element
    rows, pitch = 9, (chunks + 1) * per
    z, _ = _logits(rows, vocab, dt, vocab, pitch if on_grid else pitch + 1, 0 if on_grid else 1)
    # tokens: the first and last columns, the last whole chunk, the remainder, a chunk behind the
    # first wave's and behind a part's, a masked row
    y = torch.tensor([0, vocab - 1, chunks * per - 1, chunks * per, min(64 * per, vocab - 1),
                      min(256 * per + 1, vocab - 1), -1, vocab // 2, vocab // 3], device="cuda")
    g = torch.Generator().manual_seed(chunks)
    with _store(scale=256.0) as store:
        logps = store.token_logprobs(z, y)
        old = logps + 0.3 * torch.randn(rows, generator=g).cuda()
        ref = logps + 0.3 * torch.randn(rows, generator=g).cuda()
        adv = torch.randn(rows, generator=g).cuda()
        r = store.policy_loss(z, y, old, adv, ref, clip=(0.2, 0.3), kl_coef=0.05)
        assert torch.equal(r.logps, logps)
        only = store.policy_loss(z, y, old, adv, ref, clip=(0.2, 0.3), kl_coef=0.05, grad=False)
        for a, b in zip(r[:3], only[:3]):
            assert torch.equal(a, b)
        twin = z.clone()  # (in its place, on another row pitch)
        store.policy_loss(twin, y, old, adv, ref, clip=(0.2, 0.3), kl_coef=0.05, grad=twin)
        assert torch.equal(twin, r.grad)
    z64 = z.double().cpu().requires_grad_()
    loss, kl, logp = _policy64(z64, y, old, adv, ref, 0.2, 0.3, 0.05, None)
    (loss * 256.0).backward()
    tol = _logp_tol(z, y)
    assert ((r.logps.double().cpu() - logp).abs() <= tol).all()
    e = float(tol.max()) + 8 * U
    assert abs(float(r.loss) - loss.item()) <= 4 * e * (abs(loss.item()) + 4)
    assert abs(float(r.kl) - kl.item()) <= 4 * e * (abs(kl.item()) + 1)
    n = 8 / 256.0
    a = (adv.double().cpu() * torch.exp(logp - old.double().cpu())).abs().detach() / n
    b = 0.05 * torch.exp(ref.double().cpu() - logp).detach() / n
    c = z64.grad.abs().max(1).values
    c = torch.maximum(c, z64.grad.abs().sum(1) / 2)
    _check_grad(r.grad, z64.grad, z, c, dt, 4 * e * (a + b))
    assert (r.grad[6] == 0).all()


@pytest.mark.parametrize("limit", LIMITS[4:])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_many_rows_of_a_shape(limit, dtype):
    """Above 2048 rows the counts and sums are launches of their own: with a given denominator
    the same rows have the same bits."""
    torch = torch_mod()
    vocab = limit * (8 if dtype == "bfloat16" else 4) + 1
    z, y = _logits(2051, vocab, getattr(torch, dtype), vocab, vocab + 3, 0)
    y[::7] = -1
    v = -torch.rand(2051, device="cuda") * 9
    with _store() as store:
        r = store.policy_loss(z, y, v, v, v, kl_coef=0.1, denominator=50.0)
        few = store.policy_loss(z[2000:], y[2000:], v[2000:], v[2000:], v[2000:], kl_coef=0.1,
                                denominator=50.0)
        assert torch.equal(r.logps, store.token_logprobs(z, y))
    assert torch.equal(r.grad[2000:], few.grad) and torch.equal(r.logps[2000:], few.logps)
