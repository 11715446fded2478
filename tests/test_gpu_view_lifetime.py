"""A torch view of a store's memory keeps that memory: a store is in a cycle with its tensors, so the
collector takes it at any later allocation, and a view that outlived it would read freed pages."""
import gc
import weakref

import pytest

import block_util as B
from gpu_util import torch_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["flat", "tensor", "part"])
@pytest.mark.parametrize("mode", ["mixed", "fp32"])
def test_a_view_keeps_its_store(mode, which):
    import ttperf
    torch = torch_mod()
    store = ttperf.ParamStore([(300, 40), (40,)], mode=mode)
    store.set_stream(torch.cuda.current_stream())
    dy = torch.ones(20, 40, device="cuda", dtype=B.param_dtype(mode))
    store.accumulate_embedding_grad(0, torch.arange(20, device="cuda"), dy)
    if which == "flat":
        view = store.torch_view(ttperf.BUF_GRAD)
    elif which == "tensor":
        view = store.tensors[0].torch_view(ttperf.BUF_GRAD)
    else:  # what is made of a view shares its memory
        view = store.tensors[0].torch_view(ttperf.BUF_GRAD)[2:].reshape(-1).detach()
    there = weakref.ref(store)
    del store
    gc.collect()
    assert there() is not None  # (before its memory is touched)
    assert float(view.double().sum()) == (18 if which == "part" else 20) * 40
    del view
    gc.collect()
    assert there() is None


def test_a_closed_store_goes():
    """close() frees the memory whatever views there are; the object goes with the last of them."""
    import ttperf
    store = ttperf.ParamStore([(8,)], mode="fp32")
    view = store.torch_view(ttperf.BUF_GRAD)
    store.close()
    there = weakref.ref(store)
    del store, view
    gc.collect()
    assert there() is None
