"""Fine-tuning a small next-token model on a ParamStore: preferences first, then a policy step.

The model scores the next token from the current one: an embedding, one MLP block with a residual
connection, and an output layer.  Its forward and backward are plain products in torch on the
store's own weights; everything around them is the store's:

  * the losses give the logits' gradient, already scaled by the store's loss scale
    (preference_loss, policy_loss; token_logprobs for the reference and the rollout's scores);
  * the backward needs each linear layer's input and GELU's: they are kept in 8 bits
    (checkpoint8, gelu_checkpoint8), a quarter of fp32 or half of bf16;
  * weight and bias gradients go from the kept inputs into the store's gradient buffer
    (accumulate_linear_grad8), which AdamW steps with loss scaling and clipping.

Run: python examples/finetune.py [--steps N]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "tt-perf_amd"))
import ttperf  # noqa: E402

EMB, W1, B1, W2, B2, WO, BO = range(7)


class Model:
    """Token t -> logits of the next one: y = e + gelu(e W1 + b1) W2 + b2, e = Emb[t];
    logits = y Wo + bo."""

    def __init__(self, vocab=65, dim=96, seed=0, fmt="int8"):
        hidden = 4 * dim
        shapes = [(vocab, dim), (dim, hidden), (hidden,), (hidden, dim), (dim,), (dim, vocab),
                  (vocab,)]
        self.store = ttperf.ParamStore(shapes, mode="mixed")
        self.store.set_stream(torch.cuda.current_stream())
        self.store.configure_scaler(True, init_scale=1024.0)
        self.fmt = fmt
        gen = torch.Generator().manual_seed(seed)
        for t, s in zip(self.store.tensors, shapes):
            if len(s) == 2:
                t.set_data((torch.randn(s, generator=gen) * s[0] ** -0.5).numpy())
        # the weights the forward reads: views of the store's bf16 copies
        self.w = [t.torch_view() for t in self.store.tensors]

    def forward(self, tokens, keep=True):
        """Logits (tokens, vocab), and what the backward needs, in 8 bits."""
        store, w = self.store, self.w
        e = w[EMB][tokens]
        h = torch.addmm(w[B1], e, w[W1])
        if not keep:
            a = torch.nn.functional.gelu(h, approximate="tanh")
            y = e + torch.addmm(w[B2], a, w[W2])
            return torch.addmm(w[BO], y, w[WO]), None
        a, h8 = store.gelu_checkpoint8(h, fmt=self.fmt, approximate="tanh")
        y = e + torch.addmm(w[B2], a, w[W2])
        kept = (tokens, store.checkpoint8(e, fmt=self.fmt), h8,
                store.checkpoint8(a, fmt=self.fmt), store.checkpoint8(y, fmt=self.fmt))
        return torch.addmm(w[BO], y, w[WO]), kept

    def backward(self, grad, kept):
        """The gradients of all weights into the store, from the logits'."""
        store, w = self.store, self.w
        tokens, e8, h8, a8, y8 = kept
        store.accumulate_linear_grad8(WO, y8, grad, bias=BO)
        dy = grad @ w[WO].t().contiguous()
        store.accumulate_linear_grad8(W2, a8, dy, bias=B2)
        dh = store.gelu_backward8(h8, dy @ w[W2].t().contiguous(), approximate="tanh")
        store.accumulate_linear_grad8(W1, e8, dh, bias=B1)
        de = dy + dh @ w[W1].t().contiguous()
        demb = torch.zeros(w[EMB].shape, device=de.device)
        store.accumulate_grad(EMB, demb.index_add_(0, tokens, de.float()))


def sequences(count, length, vocab, gen):
    """Chosen sequences count up, rejected ones down, from random starts: (tokens, targets) with
    the chosen rows first; the first quarter of each is the prompt, whose targets are masked."""
    start = torch.randint(vocab, (2 * count, 1), generator=gen)
    step = torch.cat([torch.ones(count, 1), -torch.ones(count, 1)]).long()
    rows = (start + step * torch.arange(length + 1)) % vocab
    tokens, targets = rows[:, :-1], rows[:, 1:].clone()
    targets[:, :length // 4] = -100
    return tokens.reshape(-1).cuda(), targets.reshape(-1).cuda()


def preference_steps(model, steps, pairs=16, length=24, lr=3e-3, seed=1):
    """Direct preference optimisation against the model as it was; returns the losses."""
    store = model.store
    vocab = model.w[EMB].shape[0]
    opt = ttperf.AdamW(store.parameters(), lr=lr, max_grad_norm=1.0)
    gen = torch.Generator().manual_seed(seed)
    tokens, targets = sequences(pairs, length, vocab, gen)
    starts = torch.arange(0, 2 * pairs * length + 1, length, device="cuda")
    reference = store.token_logprobs(model.forward(tokens, keep=False)[0], targets)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        logits, kept = model.forward(tokens)
        r = store.preference_loss(logits, targets, starts, reference, beta=0.5, grad=logits)
        model.backward(r.grad, kept)
        opt.step()
        losses.append(r.loss)
    return torch.stack(losses).tolist()


def policy_steps(model, steps, rows=512, lr=1e-3, seed=2):
    """Rollouts of one token, rewarded where it is even; returns the rewards' means."""
    store = model.store
    vocab = model.w[EMB].shape[0]
    opt = ttperf.AdamW(store.parameters(), lr=lr, max_grad_norm=1.0)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    means = []
    for _ in range(steps):
        tokens = torch.randint(vocab, (rows,), generator=gen, device="cuda")
        logits, _ = model.forward(tokens, keep=False)
        noise = torch.rand(logits.shape, generator=gen, device="cuda").clamp_(min=1e-9)
        actions = (logits.float() - (-noise.log()).log()).argmax(1)  # a sample of the softmax
        old = store.token_logprobs(logits, actions)
        reward = (actions % 2 == 0).float()
        advantage = reward - reward.mean()
        for _ in range(2):  # two updates on a rollout: the second one's ratios are not 1
            opt.zero_grad()
            logits, kept = model.forward(tokens)
            r = store.policy_loss(logits, actions, old, advantage, old, clip=(0.2, 0.28),
                                  kl_coef=0.01, grad=logits)
            model.backward(r.grad, kept)
            opt.step()
        means.append(reward.mean())
    return torch.stack(means).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=40)
    args = ap.parse_args()
    model = Model()
    losses = preference_steps(model, args.steps)
    print(f"preference loss {losses[0]:.4f} -> {losses[-1]:.4f} in {args.steps} steps")
    rewards = policy_steps(model, args.steps)
    print(f"policy reward {rewards[0]:.3f} -> {rewards[-1]:.3f} in {args.steps} rollouts")
    model.store.close()


if __name__ == "__main__":
    main()
