"""GPU tests that autograd sees what an operator writes: a tensor that torch's backward still needs
cannot be overwritten without a word."""
import pytest

from gpu_util import torch_mod
from test_gpu_losses import _store

pytestmark = pytest.mark.gpu


def test_every_given_result_is_a_new_version():
    torch = torch_mod()
    z = torch.randn(6, 40, device="cuda")
    y = torch.randint(40, (6,), device="cuda")
    v = -torch.rand(6, device="cuda")
    starts = torch.tensor([0, 3, 6], device="cuda")
    read = [t._version for t in (z, y, v, starts)]
    with _store() as store:
        def written(call, *tensors):
            before = [t._version for t in tensors]
            call()
            assert all(t._version > b for t, b in zip(tensors, before))
        t = store.token_logprobs(z, y)
        written(lambda: store.token_logprobs(z, y, out=t), t)
        p = store.preference_loss(z, y, starts)
        written(lambda: store.preference_loss(z, y, starts, out=p), *p)
        r = store.policy_loss(z, y, v, v)
        written(lambda: store.policy_loss(z, y, v, v, out=r), *r)
        for loss in (lambda g: store.preference_loss(z, y, starts, grad=g),
                     lambda g: store.policy_loss(z, y, v, v, grad=g)):
            g = torch.empty_like(z)
            written(lambda: loss(g), g)
            wide = torch.empty(6, 80, device="cuda")  # through a view: the base's version
            written(lambda: loss(wide[:, 40:]), wide)
        x = torch.randn(6, 40, device="cuda")
        kept = store.checkpoint8(x)
        written(lambda: store.checkpoint8(x, out=kept), kept.values, kept.scales)
        back = store.restore8(kept)
        written(lambda: store.restore8(kept, out=back), back)
        written(lambda: store.gelu_checkpoint8(x, out=back, kept=kept), back, kept.values,
                kept.scales)
        written(lambda: store.gelu_backward8(kept, x, out=back), back)
        # what is read keeps its version, and so does what a refused call would have written
        assert [t._version for t in (z, y, v, starts)] == read
        version = back._version
        with pytest.raises(ValueError):
            store.gelu_backward8(kept, x[:5], out=back)
        assert back._version == version


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_a_saved_result_is_not_overwritten_silently(kind):
    """A soft cap's tanh keeps its result for its backward: with the gradient in the logits' place
    torch refuses, with a tensor of its own it goes through.  A product does not keep its result:
    there the logits' place is fine."""
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(1)
    e = torch.randn(6, 8, generator=g, device="cuda")
    w = torch.randn(8, 40, generator=g, device="cuda", requires_grad=True)
    y = torch.randint(40, (6,), generator=g, device="cuda")
    v = -torch.rand(6, generator=g, device="cuda")
    starts = torch.tensor([0, 3, 6], device="cuda")
    with _store() as store:
        def loss(z, grad):
            if kind == "policy":
                return store.policy_loss(z, y, v, -v, grad=grad)
            return store.preference_loss(z, y, starts, grad=grad)
        z = torch.tanh(e @ w)
        r = loss(z, z)
        with pytest.raises(RuntimeError):
            z.backward(r.grad)
        z = torch.tanh(e @ w)
        z.backward(loss(z, True).grad)
        assert w.grad.isfinite().all() and w.grad.any()
        grads = []
        for place in (True, False):
            w.grad = None
            z = e @ w
            z.backward(loss(z, z if place else True).grad)
            grads.append(w.grad)
        assert torch.equal(*grads)


def test_gelu_in_its_inputs_place():
    torch = torch_mod()
    x = torch.randn(6, 40, device="cuda", requires_grad=True)
    with _store() as store:
        s = torch.sigmoid(x)
        store.gelu_checkpoint8(s, out=s)
        with pytest.raises(RuntimeError):
            s.sum().backward()


def test_inference_tensors_are_written():
    """They have no version to raise."""
    torch = torch_mod()
    with torch.inference_mode(), _store() as store:
        z = torch.randn(6, 40, device="cuda")
        y = torch.randint(40, (6,), device="cuda")
        want = store.token_logprobs(z, y)
        out = torch.zeros(6, device="cuda")
        assert store.token_logprobs(z, y, out=out) is out and torch.equal(out, want)
