"""GPU tests of which per-row tensors a loss takes: of the logits' row shape, flat, or with some
dimensions of it split or merged; never of another shape with as many elements, whose rows would be
paired wrongly."""
import pytest

from gpu_util import torch_mod
from test_gpu_losses import _store

pytestmark = pytest.mark.gpu
B, T, V = 4, 6, 33


def _inputs():
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(B, T, V, generator=g, device="cuda")
    y = torch.randint(V, (B, T), generator=g, device="cuda")
    v = -torch.rand(B, T, generator=g, device="cuda") * 5
    return z, y, v, torch.arange(0, B * T + 1, T, device="cuda")


def test_rows_in_another_order_are_refused():
    z, y, v, starts = _inputs()
    yt, vt = y.t().contiguous(), v.t().contiguous()
    with _store() as store:
        for call in (
                lambda: store.token_logprobs(z, yt),
                lambda: store.preference_loss(z, yt, starts),
                lambda: store.preference_loss(z, y, starts, vt),
                lambda: store.preference_loss(z.view(-1, V), y, starts, vt),
                lambda: store.policy_loss(z, yt, v, v),
                lambda: store.policy_loss(z, y, vt, v),
                lambda: store.policy_loss(z, y, v, vt),
                lambda: store.policy_loss(z, y, v, v, vt),
                lambda: store.policy_loss(z.view(-1, V), y.view(-1), v, vt)):
            with pytest.raises(ValueError):
                call()


def test_the_same_rows_in_other_dimensions_are_taken():
    torch = torch_mod()
    z, y, v, starts = _inputs()
    with _store() as store:
        want = store.policy_loss(z, y, v, v * 0.5, v)
        flat = [t.reshape(-1) for t in (y, v, v * 0.5, v)]
        for logits, rows in ((z, flat), (z.view(-1, V), flat),
                             (z.view(-1, V), [t.view(B, T) for t in flat]),
                             (z, [t.view(B, T, 1) for t in flat]),
                             (z, [t.view(2, 2, T) for t in flat]),
                             (z.view(2, 2, T, V), [t.view(B, T) for t in flat]),
                             (z.view(B, 1, T, V), [flat[0]] + [t.view(B, T) for t in flat[1:]]),
                             (z.view(-1, V), [t.view(-1, 1) for t in flat])):
            r = store.policy_loss(logits, *rows)
            assert r.logps.shape == rows[0].shape and r.grad.shape == logits.shape
            assert torch.equal(r.grad.view(-1), want.grad.view(-1))
            assert torch.equal(r.logps.view(-1), want.logps.view(-1))
            p = store.preference_loss(logits, rows[0], starts, rows[1])
            assert torch.equal(p.logps.view(-1), want.logps.view(-1))
        one = store.token_logprobs(z[0, 0], y[0, 0])
        assert one.shape == () and one == want.logps[0, 0]
        assert store.token_logprobs(z[0, 0], y[0, :1]).shape == (1,)
        none = torch.empty(0, 5, V, device="cuda")
        assert store.token_logprobs(none, y[:0]).shape == (0, T)
