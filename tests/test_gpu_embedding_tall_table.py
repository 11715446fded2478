"""The gradient of few tokens into a table whose rows take more than one launch."""
import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [2 ** 29 + 1003, 2 ** 28 + 1])
def test_few_tokens_of_a_tall_table(vocab):
    import ttperf
    torch = torch_mod()
    with ttperf.ParamStore([(vocab, 1)], mode="bf16") as store:
        store.set_stream(torch.cuda.current_stream())
        grad = B.grad(store, 0).view(-1)
        grad.fill_(3.0)
        # both sides of the launches' borders, a token twice (of 2^28 + 1 rows 2^28 is the last one: two
        # of it), two outside the table
        at = [0, vocab - 1, 2 ** 28 - 1, 2 ** 28, 7, 7, -1, vocab]
        t = torch.tensor(at, device="cuda")
        dy = torch.arange(1.0, 9.0, device="cuda").bfloat16().view(8, 1)
        named = sorted({k for k in at if 0 <= k < vocab})
        want = [sum(i + 1 for i, k in enumerate(at) if k == n) for n in named]
        store.accumulate_embedding_grad(0, t, dy)
        assert grad[torch.tensor(named, device="cuda")].tolist() == want
        assert int(torch.count_nonzero(grad)) == len(named)
        store.accumulate_embedding_grad(0, t, dy)  # added to: the other rows stay
        assert grad[torch.tensor(named, device="cuda")].tolist() == [2 * v for v in want]
        assert int(torch.count_nonzero(grad)) == len(named)
        store.zero_grad()
        grad.fill_(3.0)
        store.accumulate_embedding_grad(0, t[6:], dy[6:])  # nothing but tokens outside
        assert int(torch.count_nonzero(grad)) == 0
