"""GPU tests of the preference loss where a token has probability 0: its log-probability is -inf, the
pair's margin +inf or -inf."""
import math

import pytest

from gpu_util import torch_mod
from test_gpu_losses import _check_grad, _logits, _logp64, _logp_tol, _store, U

pytestmark = pytest.mark.gpu
BETA = 0.13


def _call(pairs, vocab, dtype, sequence, eps, scale=0.0):
    """A loss of sequences of two rows whose second row of `sequence` has a ruled-out token; the
    finite rows' logits."""
    torch = torch_mod()
    rows = 4 * pairs
    z, y = _logits(rows, vocab, dtype, vocab + pairs)
    row = 2 * sequence + 1
    z[row, y[row]] = -math.inf
    starts = torch.arange(0, rows + 1, 2, device="cuda")
    with _store(scale=scale) as store:
        r = store.preference_loss(z, y, starts, beta=BETA, label_smoothing=eps)
    return z, y, row, r


# 3 pairs are finished in the launch that scores the rows, 17 by one of their own; rows of 9000
# are scored in parts
@pytest.mark.parametrize("pairs", [3, 17])
@pytest.mark.parametrize("vocab", [65, 9000])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_rejected_token_of_probability_0(pairs, vocab, dtype):
    """Its pair is decided: margin +inf, loss -log sigmoid(+inf) = 0, gradient 0; the other pairs
    are as ever."""
    torch = torch_mod()
    z, y, row, r = _call(pairs, vocab, getattr(torch, dtype), pairs + 1, 0.0)
    rows = torch.arange(4 * pairs)
    decided = (rows // 2 == 1) | (rows // 2 == pairs + 1)
    z64 = z.double().cpu()
    z64[row] = 0  # (any finite row: it does not count)
    z64.requires_grad_()
    d = _logp64(z64, y).view(-1, 2).sum(1)
    h = BETA * (d[:pairs] - d[pairs:])
    others = torch.arange(pairs) != 1
    loss = -torch.nn.functional.logsigmoid(h[others]).sum() / pairs
    loss.backward()
    tol = _logp_tol(z64, y)
    h_tol = BETA * float(tol.sum()) + 2 * U * float(h.detach().abs().max()) + 1e-12
    m = r.margins.double().cpu()
    assert m[1] == math.inf and ((m - h.detach()).abs() <= h_tol)[others].all()
    assert r.logps[row] == -math.inf
    assert abs(float(r.loss) - loss.item()) <= h_tol + 2 * U * loss.item()
    assert (r.grad.cpu()[decided] == 0).all()
    want = z64.grad.clone()
    want[decided] = 0
    coef = want.abs().max(1).values * 2
    _check_grad(r.grad, want, z64, coef, z.dtype, coef * (h_tol + 4 * U))


@pytest.mark.parametrize("pairs", [3, 17])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_chosen_token_of_probability_0(pairs, dtype):
    """Margin -inf, loss +inf; the gradient's factor is -beta / pairs, sigmoid being 0."""
    torch = torch_mod()
    z, y, row, r = _call(pairs, 65, getattr(torch, dtype), 1, 0.0, 64.0)
    assert r.margins[1] == -math.inf and float(r.loss) == math.inf
    assert r.grad.isfinite().all()
    c = 64.0 * -BETA / pairs
    # of the token itself: c (1 - 0), one rounding of c and one to the type
    at = float(r.grad[row, y[row]])
    assert abs(at - c) <= abs(c) * (2.0 ** -8 if dtype == "bfloat16" else 2 * U)


@pytest.mark.parametrize("pairs", [3, 17])
def test_smoothing_makes_a_decided_pair_infinitely_bad(pairs):
    """With smoothing the other order has a weight too: loss +inf at either infinite margin."""
    torch = torch_mod()
    for sequence, sign in ((1, -1), (pairs + 1, 1)):
        _, _, _, r = _call(pairs, 65, torch.float32, sequence, 0.1)
        assert float(r.margins[1]) == sign * math.inf and float(r.loss) == math.inf
        assert r.grad.isfinite().all()
