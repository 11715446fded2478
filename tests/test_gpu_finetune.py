"""GPU tests of the fine-tuning operators together, in the example program: its gradients against
a 64-bit forward and backward on the kept activations' values, and its training."""
import os
import subprocess
import sys

import pytest

from conftest import REPO
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(REPO, "examples"))


def test_the_examples_gradients():
    """Every weight's gradient of one preference step, against automatic differentiation of the
    model and the loss in 64 bits from the same bf16 weights.  The kept activations differ from
    the whole ones by at most 2^-7 of their block's largest value each, the products round to bf16
    (2^-8) at six places: gradients agree to a few percent of their norm."""
    torch = torch_mod()
    import finetune
    model = finetune.Model(vocab=37, dim=40, seed=3)
    gen = torch.Generator().manual_seed(5)
    tokens, targets = finetune.sequences(5, 11, 37, gen)
    starts = torch.arange(0, 111, 11, device="cuda")
    logits, kept = model.forward(tokens)
    store = model.store
    ref = store.token_logprobs(logits, targets) + 0.1
    r = store.preference_loss(logits, targets, starts, ref, beta=0.5, label_smoothing=0.1)
    model.backward(r.grad, kept)

    w = [t.detach().double().cpu().requires_grad_() for t in model.w]
    t, y = tokens.cpu(), targets.cpu()
    e = w[0][t]
    a = torch.nn.functional.gelu(e @ w[1] + w[2], approximate="tanh")
    z = (e + a @ w[3] + w[4]) @ w[5] + w[6]
    lp = torch.log_softmax(z, 1).gather(1, y.clamp(min=0)[:, None])[:, 0]
    d = torch.where(y >= 0, lp - ref.double().cpu(), torch.zeros((), dtype=torch.float64))
    total = d.view(10, 11).sum(1)
    h = 0.5 * (total[:5] - total[5:])
    sig = torch.nn.functional.logsigmoid
    loss = (-0.9 * sig(h) - 0.1 * sig(-h)).mean()
    (loss * 1024.0).backward()  # the store's loss scale
    assert abs(float(r.loss) - loss.item()) < 0.02
    for i, want in enumerate(w):
        got = torch.from_numpy(store.tensors[i].grad.numpy()).double()
        off = float((got - want.grad).norm() / want.grad.norm())
        assert off < 0.05, (i, off)
    store.close()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_the_example_learns(fmt):
    torch_mod()
    import finetune
    model = finetune.Model(fmt=fmt)
    losses = finetune.preference_steps(model, 30)
    assert abs(losses[0] - 0.6931) < 1e-3 and losses[-1] < 0.05, losses
    rewards = finetune.policy_steps(model, 25)
    assert rewards[-1] > rewards[0] + 0.15, rewards
    model.store.close()


def test_the_example_runs():
    out = subprocess.run([sys.executable, os.path.join(REPO, "examples", "finetune.py"), "--steps",
                          "5"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "preference loss 0.6931" in out.stdout and "policy reward" in out.stdout
