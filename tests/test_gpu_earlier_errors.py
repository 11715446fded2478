"""An error that an earlier HIP call of the host left behind is not an operator's."""
import ctypes as C

import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu


def _hip():
    """The HIP runtime that this process has loaded."""
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64.so" in line)
    return C.CDLL(path)


def test_no_operator_reports_an_earlier_error():
    import ttperf
    torch = torch_mod()
    wrong = 10 ** 6  # (no such device: an error of the host call alone)
    x = torch.randn(700, 16, device="cuda")
    t = torch.arange(700, device="cuda") % 30
    w = torch.randn(30, 16, device="cuda")
    with B.store_of([w, w[0].clone(), w[1].clone()], "fp32") as store:
        hip = _hip()
        r = store.layer_norm(2, x, bias=3)
        none = store.layer_norm(2, x[:0], bias=3)
        y, dx = store.embedding(1, t), torch.empty_like(x)
        z = store.linear(1, x, transposed=True)
        store.zero_grad()
        calls = {
            "embedding": lambda: store.embedding(1, t, out=y),
            "gradient": lambda: store.accumulate_embedding_grad(1, t, x),
            "gradient of few": lambda: store.accumulate_embedding_grad(1, t[:9], x[:9]),
            "layer norm": lambda: store.layer_norm(2, x, bias=3, out=r),
            "backward": lambda: store.layer_norm_backward(2, x, x, r.mean, r.rstd, bias=3, out=dx),
            "backward of no rows": lambda: store.layer_norm_backward(
                2, x[:0], x[:0], none.mean, none.rstd, bias=3, out=dx[:0]),
            "dropout": lambda: store.dropout(x, 0.5, 1, out=dx),
            "linear": lambda: store.linear(1, x, transposed=True, out=z),
        }
        for name, call in calls.items():
            assert hip.hipSetDevice(wrong) != 0
            try:
                call()
            except ttperf.TTPError as e:
                pytest.fail(f"{name}: {e}")
            finally:
                hip.hipGetLastError()
        torch.cuda.synchronize()
