"""GPU tests of the formats a checkpoint of the caller's own memory may have."""
import pytest

from gpu_util import torch_mod
from test_gpu_checkpoint8 import _store

pytestmark = pytest.mark.gpu


def test_a_checkpoint_of_an_unknown_format():
    import ttperf
    torch = torch_mod()
    with _store() as store:
        kept = store.checkpoint8(torch.randn(6, 64, device="cuda"))
        with pytest.raises(ValueError):
            ttperf.Checkpoint8(kept.values, kept.scales, (6, 64), torch.float32, "int4")
