"""GPU tests of the tensors that linear gradients from 8-bit inputs may go to."""
import pytest

from gpu_util import torch_mod
from test_gpu_linear_grad8 import _inputs, _store

pytestmark = pytest.mark.gpu


def test_tensors_that_do_not_exist():
    """An index is a tensor's number, whatever it would be in 32 bits: -1 is no "no bias"."""
    torch = torch_mod()
    x, dy = _inputs(20, 40, 24, torch.bfloat16, 5)
    with _store(40, 24) as store:
        kept = store.checkpoint8(x)
        for index, bias in ((1, -1), (1, 4), (1, 2 ** 32 + 2), (-3, 2), (4, 2),
                            (2 ** 32 + 1, 2), (1, -2)):
            with pytest.raises(ValueError):
                store.accumulate_linear_grad8(index, kept, dy, bias=bias)
            assert not any(store.has_grad(i) for i in range(4))
        store.accumulate_linear_grad8(1, kept, dy, bias=2)
        assert [store.has_grad(i) for i in range(4)] == [False, True, True, False]
