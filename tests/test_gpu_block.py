"""GPU tests of a block's operators together: a small pre-norm language model on a store (token and
position embeddings, dropout, layer norm, an MLP with GELU, dropout and a residual, a tied output
layer, the policy loss), its gradients against automatic differentiation in 64 bits, and one step
captured into a graph."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu
VOCAB, DIM, CONTEXT, LAYERS, P = 67, 40, 16, 2, 0.2
WTE, WPE, LNF, LNF_B = 0, 1, 2, 3
FIRST, EACH = 4, 6  # a block's: ln weight, bias, W1, b1, W2, b2


def _shapes():
    block = [(DIM,), (DIM,), (DIM, 4 * DIM), (4 * DIM,), (4 * DIM, DIM), (DIM,)]
    return [(VOCAB, DIM), (CONTEXT, DIM), (DIM,), (DIM,)] + block * LAYERS


def _store(mode, seed=0):
    import ttperf
    torch = torch_mod()
    store = ttperf.ParamStore(_shapes(), mode=mode)
    store.set_stream(torch.cuda.current_stream())
    g = torch.Generator().manual_seed(seed)
    for i, (t, s) in enumerate(zip(store.tensors, _shapes())):
        w = torch.randn(s, generator=g) * (s[0] ** -0.5 if len(s) == 2 and i > 1 else 0.3)
        t.set_data((w + (1 if i == LNF or (i >= FIRST and (i - FIRST) % EACH == 0) else 0)).numpy())
    return store


class Results:
    """Results by the order of the calls: new ones in a first pass, written again in later ones."""

    def __init__(self):
        self.kept, self.at = [], None

    def start(self, again):
        self.at = 0 if again else None

    def __call__(self, call, *args, out="out", **kwargs):
        if self.at is None:
            r = call(*args, **kwargs)
            self.kept.append(r)
            return r
        kwargs[out] = self.kept[self.at]
        if out == "gelu":
            kwargs["out"], kwargs["kept"] = kwargs.pop("gelu")
        self.at += 1
        return call(*args, **kwargs)


def _step(store, data, seed, r):
    """Forward, loss and backward: the gradients go to the store."""
    tokens, positions, targets, old, adv = data
    kept = []
    x = r(store.embedding, WTE, tokens, position=WPE, positions=positions)
    x = r(store.dropout, x, P, seed)
    for k in range(LAYERS):
        at = FIRST + k * EACH
        n = r(store.layer_norm, at, x, bias=at + 1)
        h = r(store.linear, at + 2, n.y, bias=at + 3)
        a, h8 = r(store.gelu_checkpoint8, h, approximate="tanh", out="gelu")
        kept.append((x, n, r(store.checkpoint8, n.y), h8, r(store.checkpoint8, a)))
        x = r(store.linear, at + 4, a, bias=at + 5, dropout=(P, seed, k + 1), residual=x)
    n = r(store.layer_norm, LNF, x, bias=LNF_B)
    last8 = r(store.checkpoint8, n.y)
    z = r(store.linear, WTE, n.y, transposed=True)
    loss = r(store.policy_loss, z, targets, old, adv, kl_coef=0.0)

    store.accumulate_linear_grad8(WTE, last8, loss.grad, transposed=True)
    d = r(store.linear_input_grad, WTE, loss.grad, transposed=True)
    d = r(store.layer_norm_backward, LNF, x, d, n.mean, n.rstd, bias=LNF_B)
    for k in reversed(range(LAYERS)):
        at = FIRST + k * EACH
        x, n, y8, h8, a8 = kept[k]
        dm = r(store.dropout, d, P, seed, stream=k + 1)
        store.accumulate_linear_grad8(at + 4, a8, dm, bias=at + 5)
        dh = r(store.gelu_backward8, h8, r(store.linear_input_grad, at + 4, dm),
               approximate="tanh")
        store.accumulate_linear_grad8(at + 2, y8, dh, bias=at + 3)
        d = r(store.layer_norm_backward, at, x, r(store.linear_input_grad, at + 2, dh), n.mean,
              n.rstd, bias=at + 1, add=d)
    d = r(store.dropout, d, P, seed)
    store.accumulate_embedding_grad(WTE, tokens, d)  # behind the output layer's
    store.accumulate_embedding_grad(WPE, positions, d)
    return loss, kept, last8


def _data(seed, rows=48):
    torch = torch_mod()
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(VOCAB, (rows,), generator=g, device="cuda")
    tokens[5] = -1  # padding
    targets = torch.randint(VOCAB, (rows,), generator=g, device="cuda")
    targets[::7] = -100
    positions = torch.arange(rows, device="cuda") % CONTEXT
    old = -4.2 + 0.1 * torch.randn(rows, generator=g, device="cuda")
    return tokens, positions, targets, old, torch.randn(rows, generator=g, device="cuda")


def _reference(store, w, data, seed, kept, y8):
    """The loss in 64 bits.  Where the operators' backward takes an input from 8 bits, so does this
    one's: the value is the whole input's, the gradient the kept one's."""
    torch = torch_mod()
    tokens, positions, targets, old, adv = [t.cpu() for t in data]

    def whole(c):
        return store.restore8(c, dtype=torch.float32).double().cpu().reshape(c.shape)

    def linear(x, x8, m):
        k = whole(x8)
        return x @ m.detach() + (k @ m - (k @ m).detach())

    def gelu(h, h8):
        g = torch.nn.functional.gelu(whole(h8) + h - h.detach(), approximate="tanh")
        return torch.nn.functional.gelu(h, approximate="tanh").detach() + g - g.detach()

    def drop(x, stream):
        keep = torch.from_numpy(B.kept(*x.shape, P, seed, stream))
        t = B.threshold(P)
        return torch.where(keep, x * (65536 / (65536 - t)), torch.zeros((), dtype=torch.float64))

    def norm(x, i):
        return torch.nn.functional.layer_norm(x, (DIM,), w[i], w[i + 1], 1e-5)

    e = torch.where((tokens >= 0)[:, None], w[WTE][tokens.clamp(min=0)],
                    torch.zeros((), dtype=torch.float64))
    x = drop(e + w[WPE][positions], 0)
    for k in range(LAYERS):
        at = FIRST + k * EACH
        _, _, n8, h8, a8 = kept[k]
        h = linear(norm(x, at), n8, w[at + 2]) + w[at + 3]
        x = x + drop(linear(gelu(h, h8), a8, w[at + 4]) + w[at + 5], k + 1)
    z = linear(norm(x, LNF), y8, w[WTE].t())
    lp = torch.log_softmax(z, 1).gather(1, targets.clamp(min=0)[:, None])[:, 0]
    live, adv = targets >= 0, adv.double()
    ratio = torch.exp(lp - old.double())
    loss = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)
    return torch.where(live, loss, torch.zeros((), dtype=torch.float64)).sum() / live.sum()


@pytest.mark.parametrize("mode,bound", [("fp32", 1e-4), ("mixed", 0.06)])
def test_gradients(mode, bound):
    """Relative in norm.  fp32: about thirty operators one behind the other, of sums of at most 160
    numbers, each within (160 / 16 + 64) u < 5e-6 of its terms' magnitudes, of which the results are
    no less than a third.  mixed: as many roundings to bf16, 2^-8 each, not one direction's."""
    torch = torch_mod()
    store = _store(mode)
    for seed in (1, 2 ** 40 + 3):
        data = _data(seed)
        store.zero_grad()
        loss, kept, last8 = _step(store, data, seed, Results())
        w = [t.torch_view().detach().double().cpu().reshape(s).requires_grad_()
             for t, s in zip(store.tensors, _shapes())]
        want = _reference(store, w, data, seed, kept, last8)
        want.backward()
        assert abs(float(loss.loss) - want.item()) <= bound * max(1.0, abs(want.item()))
        for i, t in enumerate(store.tensors):
            got = t.torch_view(_grad()).double().cpu().reshape(_shapes()[i])
            off = float((got - w[i].grad).norm() / w[i].grad.norm())
            assert off < bound, (i, off)
    store.close()


def _grad():
    import ttperf
    return ttperf.BUF_GRAD


def test_one_step_captured():
    """The whole step with its zero_grad in a graph, the seed on the device: each launch gives what
    the eager step gives, with other work between them."""
    torch = torch_mod()
    store = _store("mixed")
    seed = torch.tensor([7], device="cuda")
    data = _data(3)
    store.set_stream(torch.cuda.Stream())
    torch.cuda.synchronize()
    r = Results()
    _step(store, data, seed, r)
    r.start(True)
    store.begin_capture()
    store.zero_grad(set_to_none=True)
    loss, _, _ = _step(store, data, seed, r)
    graph = store.end_capture()
    for k in range(4):
        for t, new in zip(data, _data(20 + k)):
            t.copy_(new)
        seed.fill_(100 + k)
        torch.cuda.synchronize()
        graph.replay()
        store.sync()
        got = [store.torch_view(_grad()).clone(), loss.loss.clone(), loss.grad.clone()]
        store.zero_grad(set_to_none=True)
        e, _, _ = _step(store, data, 100 + k, Results())
        torch.cuda.synchronize()
        for u, v in zip(got, (store.torch_view(_grad()), e.loss, e.grad)):
            assert torch.equal(u, v)
        assert got[0].abs().sum() > 0
    graph.close()
    store.close()


def test_steps_with_loss_scaling():
    """A few AdamW steps run with loss scaling, and every gradient stays finite."""
    import ttperf
    torch = torch_mod()
    store = _store("mixed")
    store.configure_scaler(True, init_scale=256.0)
    opt = ttperf.AdamW(store.parameters(), lr=1e-3, max_grad_norm=1.0)
    for k in range(5):
        opt.zero_grad()
        loss, _, _ = _step(store, _data(k), k, Results())
        assert store.torch_view(_grad()).isfinite().all() and loss.loss.isfinite()
        opt.step()
    assert store.step_count == 5
    store.close()
